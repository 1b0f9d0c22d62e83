"""Calls whose rows choose their own weights, as a server of many adapters, their trainer and a mixture of experts make them:

* ``forward``   a packed projection with a low-rank adapter of each row's own out of a bank
* ``backward``  its gradients: of the rows, and of every adapter of the bank
* ``experts``   a mixture-of-experts MLP of packed projections for a few tokens
* ``route``     the choice of those experts: softmax and the largest of a row's logits

Packed weights are in the layout that the library documents: chunks of 16 columns x 128 rows, ``[column tile][group]``, 256 words
each; word ``4 * lane + t`` of a chunk belongs to column ``lane % 16`` and holds rows ``32 t + 8 (lane // 16) + j``, row ``j`` in
nibble ``j // 2 + 4 * (j % 2)``; scales ``[column tile][group][16]``.  Value = (code - 8) * scale."""
import math

import torch

own = False

DEVICE = "cuda"
NIBBLE = (0, 4, 1, 5, 2, 6, 3, 7)      # of row j inside a word


# ---- the cases -------------------------------------------------------------------------------------------------

def listed():
    return [
        # one request decodes: the smallest call, the square projection of the smallest configuration
        {"name": "forward 1 row", "op": "forward", "m": 1, "k": 2560, "n": 2560, "g": 128, "count": 4, "rank": 8, "requests": 1, "bare": 0},
        # a decode step of sixteen requests with an adapter each, the fused gate+up projection
        {"name": "forward 16 rows", "op": "forward", "m": 16, "k": 2560, "n": 18432, "g": 128, "count": 32, "rank": 16, "requests": 16, "bare": 0},
        # decodes and short prompts side by side, some without an adapter, the down projection, a rank that is no power of two
        {"name": "forward 77 rows", "op": "forward", "m": 77, "k": 9216, "n": 2560, "g": -1, "count": 9, "rank": 24, "requests": 23, "bare": 3},
        # a prefill of several prompts at once
        {"name": "forward 2048 rows", "op": "forward", "m": 2048, "k": 2560, "n": 18432, "g": 128, "count": 8, "rank": 32, "requests": 7, "bare": 1},
        # a training step on a few short texts, the output projection of an attention layer
        {"name": "backward 45 rows", "op": "backward", "m": 45, "k": 4096, "n": 2560, "g": 128, "count": 2, "rank": 8, "requests": 3, "bare": 0},
        # ragged texts of several adapters, the down projection
        {"name": "backward 777 rows", "op": "backward", "m": 777, "k": 9216, "n": 2560, "g": 128, "count": 6, "rank": 16, "requests": 11, "bare": 1},
        # a full training step of four adapters, the fused gate+up projection
        {"name": "backward 2048 rows", "op": "backward", "m": 2048, "k": 2560, "n": 18432, "g": 128, "count": 4, "rank": 32, "requests": 8, "bare": 0},
        # one request decodes
        {"name": "experts 1 token", "op": "experts", "m": 1, "k": 2560, "n": 1024, "g": 128, "experts": 64, "top": 8, "away": 0},
        # a handful of requests, experts with scales per column, a quarter of the experts on another GPU
        {"name": "experts 13 tokens", "op": "experts", "m": 13, "k": 2048, "n": 1280, "g": -1, "experts": 32, "top": 4, "away": 8},
        # a decode step of 64 requests: nearly every expert has rows
        {"name": "experts 64 tokens", "op": "experts", "m": 64, "k": 2560, "n": 1024, "g": 128, "experts": 64, "top": 8, "away": 0},
        # one request decodes
        {"name": "route 1 row", "op": "route", "m": 1, "experts": 64, "top": 8, "renormalise": True, "dtype": "bfloat16", "masked": 0},
        # the prompts of a prefill
        {"name": "route 8192 rows", "op": "route", "m": 8192, "experts": 128, "top": 8, "renormalise": True, "dtype": "float32", "masked": 5},
    ]


def _spread(rng, low, high, step=1):
    """Of low, low + step, ... high, even over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + step)))
    return max(low, min(high, int(v) // step * step))


def draw(rng):
    op = rng.choice(("forward", "forward", "backward", "experts", "route"))
    if op == "route":
        experts = _spread(rng, 4, 512)
        return {"op": op, "m": _spread(rng, 1, 8192), "experts": experts, "top": rng.randint(1, min(16, experts)),
                "renormalise": rng.random() < 0.5, "dtype": rng.choice(("bfloat16", "float16", "float32")),
                "masked": rng.randint(0, experts // 4)}
    if op == "experts":
        experts = _spread(rng, 4, 64)
        return {"op": op, "m": _spread(rng, 1, 64), "k": _spread(rng, 256, 2560, 256), "n": _spread(rng, 256, 1024, 128),
                "g": rng.choice((128, 128, -1)), "experts": experts, "top": rng.randint(1, min(8, experts)), "away": rng.randint(0, experts // 4)}
    m = _spread(rng, 1, 2048)
    requests = rng.randint(1, min(m, 64))
    return {"op": op, "m": m, "k": _spread(rng, 256, 9216, 128), "n": _spread(rng, 256, 5120, 256), "g": rng.choice((128, 128, -1)),
            "count": rng.randint(1, 16), "rank": 8 * rng.randint(1, 4), "requests": requests, "bare": rng.randint(0, requests // 3)}


# ---- inputs ----------------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(shape, device=DEVICE, generator=gen)


def _codes(gen, *shape):
    """Words of eight codes of rounded normal weights, as quantising gives them."""
    words = torch.zeros(shape, dtype=torch.int32, device=DEVICE)
    for j in range(8):
        words |= (_normal(gen, *shape) * 2.3 + 8).round_().clamp_(0, 15).to(torch.int32) << 4 * j
    return words


def _weight(gen, k, n, g, *lead):
    """A packed weight and its scales: entries of about 1 / sqrt(k)."""
    scales = (torch.rand((*lead, 1 if g == -1 else k // g, n), device=DEVICE, generator=gen) * 0.5 + 0.75) / (2.3 * math.sqrt(k))
    return _codes(gen, *lead, k // 16, 2 * n), scales.half()


def _rows_of_requests(gen, m, requests, bare, count):
    """The adapter of each row: `requests` runs of rows of ragged lengths, each with an adapter of its own choice, `bare` of them with none (-1)."""
    cuts = torch.randperm(m - 1, device=DEVICE, generator=gen)[:requests - 1] if m > 1 else torch.zeros(0, dtype=torch.int64, device=DEVICE)
    starts = torch.zeros(m, dtype=torch.int64, device=DEVICE)
    starts[cuts + 1] = 1
    of = torch.arange(requests, device=DEVICE) + torch.randint(0, count, (1,), device=DEVICE, generator=gen)
    of = of[torch.randperm(requests, device=DEVICE, generator=gen)] % count
    of[torch.randperm(requests, device=DEVICE, generator=gen)[:bare]] = -1
    return of[starts.cumsum(0)].to(torch.int32)


def prepare(case, seed):
    gen = _generator(seed)
    if case["op"] == "route":
        logits = _normal(gen, case["m"], case["experts"]) * 1.5
        if case["masked"]:                       # experts that this rank does not offer
            logits[:, torch.randperm(case["experts"], device=DEVICE, generator=gen)[:case["masked"]]] = -math.inf
        return {"op": "route", "logits": logits.to(getattr(torch, case["dtype"])), "top": case["top"], "renormalise": case["renormalise"]}
    m, k, n, g = case["m"], case["k"], case["n"], case["g"]
    x = _normal(gen, m, k).to(torch.bfloat16)
    if case["op"] == "experts":
        experts, top = case["experts"], case["top"]
        scores = _normal(gen, m, experts) * 1.5
        order = scores.argsort(dim=1, descending=True)[:, :top]
        weights = torch.softmax(torch.gather(scores, 1, order), dim=1)
        of = torch.where(order >= experts - case["away"], -1, order).to(torch.int32)
        b_gate_up, s_gate_up = _weight(gen, k, 2 * n, g, experts)
        b_down, s_down = _weight(gen, n, k, g, experts)
        return {"op": "experts", "x": x, "of": of, "weights": weights, "b_gate_up": b_gate_up, "s_gate_up": s_gate_up,
                "b_down": b_down, "s_down": s_down, "g": g}
    b, s = _weight(gen, k, n, g)
    count, rank = case["count"], case["rank"]
    state = {"op": case["op"], "x": x, "b": b, "s": s, "g": g,
             "bank_a": (_normal(gen, count, rank, k) / math.sqrt(k)).to(torch.bfloat16),
             "bank_b": (_normal(gen, count, n, rank) * 0.3 / math.sqrt(rank)).to(torch.bfloat16),
             "bank_scales": torch.rand(count, device=DEVICE, generator=gen) + 0.5,
             "of": _rows_of_requests(gen, m, case["requests"], case["bare"], count)}
    if case["op"] == "backward":
        state["dy"] = (_normal(gen, m, n) * 0.01).to(torch.bfloat16)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------

def run(s):
    if s["op"] == "forward":
        return _own_forward(s) if own else _forward(s)
    if s["op"] == "backward":
        return _own_backward(s) if own else _backward(s)
    if s["op"] == "experts":
        return _own_experts(s) if own else _experts(s)
    return _own_route(s) if own else _route(s)


def _own_forward(s):
    from kiln_amd import marlin_gemm
    return marlin_gemm.marlin_w4a16_gemm_bank(s["x"], s["b"], s["s"], s["g"], s["bank_a"], s["bank_b"], s["bank_scales"], s["of"])


def _own_backward(s):
    from kiln_amd import marlin_gemm
    dx, d_bank_a, d_bank_b = marlin_gemm.marlin_w4a16_gemm_bank_backward(s["dy"], s["x"], s["b"], s["s"], s["g"], s["bank_a"], s["bank_b"],
                                                                         s["bank_scales"], s["of"])
    return {"dx": dx, "d_bank_a": d_bank_a, "d_bank_b": d_bank_b}


def _own_experts(s):
    from kiln_amd import marlin_gemm
    return marlin_gemm.marlin_w4a16_moe(s["x"], s["of"], s["weights"], s["b_gate_up"], s["s_gate_up"], s["b_down"], s["s_down"], s["g"])


def _own_route(s):
    from kiln_amd import marlin_gemm
    of, weights = marlin_gemm.moe_route(s["logits"], s["top"], s["renormalise"])
    return {"of": of, "weights": weights}


def _unpacked(b, scales):
    """Packed weights [..., k/16, 2n] and their scales as float32 [..., k, n]."""
    lead, k, n = b.shape[:-2], b.shape[-2] * 16, b.shape[-1] // 2
    groups = scales.shape[-2]
    shifts = torch.tensor([4 * p for p in NIBBLE], dtype=torch.int32, device=b.device)
    words = b.reshape(-1, n // 16, k // 128, 4, 16, 4, 1)                        # column tile, group, kq, column, t
    codes = ((words >> shifts) & 15).permute(0, 2, 5, 3, 6, 1, 4)                 # group, t, kq, j, column tile, column
    w = (codes - 8).to(torch.float32).reshape(-1, groups, k // groups, n)
    s = scales.reshape(-1, n // 16, groups, 16).permute(0, 2, 1, 3).reshape(-1, groups, 1, n).to(torch.float32)
    return (w * s).reshape(*lead, k, n)


def _chosen(s):
    """[m, count * rank]: the scale of each row's own adapter in that adapter's rank columns, zero in the others'."""
    count, rank = s["bank_a"].shape[:2]
    hot = s["of"][:, None] == torch.arange(count, dtype=torch.int32, device=DEVICE)
    return (hot * s["bank_scales"])[:, :, None].expand(-1, -1, rank).reshape(-1, count * rank)


def _forward(s):
    x, k, n = s["x"].float(), s["x"].shape[1], s["s"].shape[1]
    t = (x @ s["bank_a"].float().reshape(-1, k).t()) * _chosen(s)
    y = x @ _unpacked(s["b"], s["s"]) + t @ s["bank_b"].float().transpose(1, 2).reshape(-1, n)
    return y.to(torch.bfloat16)


def _backward(s):
    x, dy, k, n = s["x"].float(), s["dy"].float(), s["x"].shape[1], s["dy"].shape[1]
    a, b = s["bank_a"].float().reshape(-1, k), s["bank_b"].float().transpose(1, 2).reshape(-1, n)
    count, rank = s["bank_a"].shape[:2]
    chosen = _chosen(s)
    u = (dy @ b.t()) * chosen
    dx = dy @ _unpacked(s["b"], s["s"]).t() + u @ a
    d_a = (u.t() @ x).reshape(count, rank, k)
    d_b = (((x @ a.t()) * chosen).t() @ dy).reshape(count, rank, n).transpose(1, 2)
    return {"dx": dx.to(torch.bfloat16), "d_bank_a": d_a.to(torch.bfloat16), "d_bank_b": d_b.to(torch.bfloat16).contiguous()}


def _experts(s):
    x, of, weights, experts = s["x"].float(), s["of"].long(), s["weights"], s["b_down"].shape[0]
    m, top = of.shape
    n = s["b_down"].shape[1] * 16
    weights = torch.where(of >= 0, weights, torch.zeros_like(weights))
    if m * top <= experts:                       # each row's own experts
        pick = of.clamp_min(0).reshape(-1)
        rows = x.repeat_interleave(top, 0)[:, None]
        b_gate_up, s_gate_up, b_down, s_down = (s[name][pick] for name in ("b_gate_up", "s_gate_up", "b_down", "s_down"))
        share = weights.reshape(-1, 1, 1)
    else:                                        # every expert over every row
        rows = x.expand(experts, -1, -1)
        b_gate_up, s_gate_up, b_down, s_down = (s[name] for name in ("b_gate_up", "s_gate_up", "b_down", "s_down"))
        share = ((of[:, :, None] == torch.arange(experts, device=DEVICE)) * weights[:, :, None]).sum(1).t()[:, :, None]
    gate_up = torch.bmm(rows, _unpacked(b_gate_up, s_gate_up)).reshape(*rows.shape[:2], n // 8, 2, 8)
    gate, up = gate_up[..., 0, :].reshape(*rows.shape[:2], n), gate_up[..., 1, :].reshape(*rows.shape[:2], n)
    y = torch.bmm(gate / (1 + torch.exp(-gate)) * up, _unpacked(b_down, s_down)) * share
    return (y.reshape(m, top, -1).sum(1) if m * top <= experts else y.sum(0)).to(torch.bfloat16)


def _route(s):
    logits = s["logits"].float()
    value, of = torch.sort(logits, dim=1, descending=True, stable=True)      # ties: the lowest index first
    value, of = value[:, :s["top"]], of[:, :s["top"]]
    top = value[:, :1]
    weights = torch.exp(value - top) / torch.exp(logits - top).sum(1, keepdim=True)
    if s["renormalise"]:
        weights = weights / weights.sum(1, keepdim=True)
    return {"of": torch.where(value == -math.inf, -1, of).to(torch.int32), "weights": weights}


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def _weight_bytes(k, n, g):
    return k * n // 2 + (1 if g == -1 else k // g) * n * 2


def work(case):
    m = case["m"]
    if case["op"] == "route":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": m * case["experts"] * size + m * case["top"] * 8, "flops": 3 * m * case["experts"]}
    k, n, g = case["k"], case["n"], case["g"]
    if case["op"] == "experts":
        here = m * case["top"] * (case["experts"] - case["away"]) / case["experts"]     # rows times experts, of those here
        used = (case["experts"] - case["away"]) * (1 - (1 - case["top"] / case["experts"]) ** m)
        return {"bytes": used * (_weight_bytes(k, 2 * n, g) + _weight_bytes(n, k, g)) + 4 * m * k + 8 * m * case["top"], "flops": here * 6 * k * n}
    used = min(case["count"], case["requests"] - case["bare"])
    low = used * case["rank"] * (k + n)
    rows = m * (case["requests"] - case["bare"]) / case["requests"]
    if case["op"] == "forward":
        return {"bytes": _weight_bytes(k, n, g) + 2 * m * (k + n) + 2 * low + 4 * m, "flops": 2 * m * k * n + 2 * rows * case["rank"] * (k + n)}
    return {"bytes": _weight_bytes(k, n, g) + 2 * m * (2 * k + n) + 2 * low + 2 * case["count"] * case["rank"] * (k + n) + 4 * m,
            "flops": 2 * m * k * n + 6 * rows * case["rank"] * (k + n)}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------

def _exact_weight(b, scales):
    """One packed weight as float64 [k, n], entry by entry from the layout's definition."""
    k, n = b.shape[0] * 16, b.shape[1] // 2
    row, col = torch.arange(k, device=DEVICE)[:, None], torch.arange(n, device=DEVICE)[None, :]
    inside = row % 128
    lane = col % 16 + 16 * (inside % 32 // 8)
    word = b.reshape(-1)[((col // 16) * (k // 128) + row // 128) * 256 + lane * 4 + inside // 32]
    j = row % 8
    code = (word.long() >> (4 * (j // 2 + 4 * (j % 2)))) & 15
    groups = scales.shape[0]
    s = scales.reshape(-1)[((col // 16) * groups + row // (k // groups)) * 16 + col % 16].double()
    return (code - 8).double() * s


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "route":
        logits = s["logits"].double().cpu()
        weights = torch.zeros(len(logits), s["top"], dtype=torch.float64)
        share, left = torch.softmax(logits, 1), logits.clone()
        for i in range(s["top"]):
            best = left.max(1, keepdim=True).values
            at = (left == best).double().argmax(1, keepdim=True)
            weights[:, i:i + 1] = torch.where(best == -math.inf, 0.0, share.gather(1, at))
            left.scatter_(1, at, -math.inf)
        return {"of": None, "weights": weights / weights.sum(1, keepdim=True) if s["renormalise"] else weights}
    x = s["x"].double()
    if s["op"] == "experts":
        y = torch.zeros_like(x)
        n = s["b_down"].shape[1] * 16
        gates = [i for i in range(2 * n) if i % 16 < 8]
        ups = [i + 8 for i in gates]
        for e in sorted(set(s["of"].reshape(-1).tolist()) - {-1}):
            rows, place = torch.nonzero(s["of"] == e, as_tuple=True)
            w = _exact_weight(s["b_gate_up"][e], s["s_gate_up"][e])
            gate, up = x[rows] @ w[:, gates], x[rows] @ w[:, ups]
            y.index_add_(0, rows, (gate * torch.sigmoid(gate) * up) @ _exact_weight(s["b_down"][e], s["s_down"][e]) * s["weights"][rows, place].double()[:, None])
        return y
    w = _exact_weight(s["b"], s["s"])
    if s["op"] == "forward":
        y = x @ w
        for i in range(len(s["bank_a"])):
            mine = s["of"] == i
            y[mine] += s["bank_scales"][i].double() * ((x[mine] @ s["bank_a"][i].double().t()) @ s["bank_b"][i].double().t())
        return y
    dy = s["dy"].double()
    dx, d_a, d_b = dy @ w.t(), torch.zeros_like(s["bank_a"], dtype=torch.float64), torch.zeros_like(s["bank_b"], dtype=torch.float64)
    for i in range(len(d_a)):
        mine, scale, a, b = s["of"] == i, s["bank_scales"][i].double(), s["bank_a"][i].double(), s["bank_b"][i].double()
        u = scale * (dy[mine] @ b)
        dx[mine] += u @ a
        d_a[i] = u.t() @ x[mine]
        d_b[i] = scale * (dy[mine].t() @ (x[mine] @ a.t()))
    return {"dx": dx, "d_bank_a": d_a, "d_bank_b": d_b}

"""What a mixture-of-experts layer on packed experts needs beyond a few tokens, to prefill a prompt and to be trained through:

* ``sort``              a router's choices in the order of their experts, and the tokens' rows in that order
* ``sort backward``     the rows' gradient back to their tokens
* ``combine``           the experts' rows back to their tokens, with the router's weights applied
* ``combine backward``  its gradients: of the rows and of the weights
* ``experts``           rows of one expert together times that expert's packed weight, as they stand or straight from the tokens, with or
                        without silu(gate) * up
* ``experts backward``  the gradient of those rows, the packed weights frozen
* ``keep``              silu(gate) * up in training: gate and up kept in 8 bits for the backward pass, and that pass out of them

A row of ``expert_of`` names a token's experts, -1 an expert held elsewhere.  Pair ``p = token * top + place`` of it has position
``place[p]`` in the sorted order, pairs of one expert together in their order, pairs without an expert last; ``order`` is the inverse, and
expert e has the positions ``first[e] ... first[e + 1]``.  Rows behind ``first[experts]`` are zero wherever they are written.

Packed weights are in the layout that the library documents: chunks of 16 columns x 128 rows, ``[column tile][group]``, 256 words
each; word ``4 * lane + t`` of a chunk belongs to column ``lane % 16`` and holds rows ``32 t + 8 (lane // 16) + j``, row ``j`` in
nibble ``j // 2 + 4 * (j % 2)``; scales ``[column tile][group][16]``.  Value = (code - 8) * scale.  Gate and up lie side by side, 8
columns of one and the 8 matching ones of the other.

Gate and up are kept as 8-bit whole numbers that share a power of two in blocks of 32 of a row's gate values, or of its up values: with e
the largest one's exponent (2^e <= |v| < 2^(e + 1), e >= -126), value = whole * 2^(e - 6), rounded to the nearest, ties to even, at most
127 in magnitude."""
import math

import torch

own = False

DEVICE = "cuda"
NIBBLE = (0, 4, 1, 5, 2, 6, 3, 7)      # of row j inside a word


# ---- the cases -------------------------------------------------------------------------------------------------

def listed():
    return [
        # one request decodes: the smallest call
        {"name": "sort 1 token", "op": "sort", "m": 1, "k": 2560, "experts": 64, "top": 8, "away": 0},
        # the prompts of a prefill, a part of the experts on another GPU
        {"name": "sort 8192 tokens", "op": "sort", "m": 8192, "k": 2048, "experts": 128, "top": 8, "away": 16},
        # a training step on a few texts
        {"name": "sort backward 1000 tokens", "op": "sort backward", "m": 1000, "k": 2560, "experts": 64, "top": 8, "away": 0},
        # a decode step of 64 requests
        {"name": "combine 64 tokens", "op": "combine", "m": 64, "k": 2560, "experts": 64, "top": 8, "away": 0},
        # a full training step
        {"name": "combine backward 4096 tokens", "op": "combine backward", "m": 4096, "k": 2560, "experts": 64, "top": 8, "away": 0},
        # a short prompt beside some decodes: a dozen rows to an expert, gate and up straight from the tokens
        {"name": "experts 96 tokens", "op": "experts", "m": 96, "k": 2560, "n": 2048, "g": 128, "experts": 64, "top": 8, "away": 0, "swiglu": True},
        # ragged prompts on experts with scales per column, a quarter of them on another GPU: the down projection
        {"name": "experts 777 tokens", "op": "experts", "m": 777, "k": 1280, "n": 2048, "g": -1, "experts": 32, "top": 4, "away": 8, "swiglu": False},
        # a prefill or training step
        {"name": "experts 2048 tokens", "op": "experts", "m": 2048, "k": 2560, "n": 2048, "g": 128, "experts": 64, "top": 8, "away": 0, "swiglu": True},
        # a training step on a few short texts, the down projection
        {"name": "experts backward 45 tokens", "op": "experts backward", "m": 45, "k": 1024, "n": 2560, "g": 128, "experts": 64, "top": 8, "away": 0},
        # a full training step, gate and up
        {"name": "experts backward 2048 tokens", "op": "experts backward", "m": 2048, "k": 2560, "n": 2048, "g": 128, "experts": 64, "top": 8, "away": 0},
        # a handful of rows of one expert
        {"name": "keep 5 rows", "op": "keep", "m": 5, "n": 1024},
        # a full training step through a dense layer
        {"name": "keep 4096 rows", "op": "keep", "m": 4096, "n": 9216},
    ]


def _spread(rng, low, high, step=1):
    """Of low, low + step, ... high, even over the logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high + step)))
    return max(low, min(high, int(v) // step * step))


def draw(rng):
    op = rng.choice(("sort", "sort backward", "combine", "combine backward", "experts", "experts", "experts backward", "experts backward", "keep"))
    if op == "keep":
        return {"op": op, "m": _spread(rng, 1, 4096), "n": _spread(rng, 128, 9216, 128)}
    experts = _spread(rng, 4, 64)
    case = {"op": op, "m": _spread(rng, 1, 2048), "experts": experts, "top": rng.randint(1, min(8, experts)), "away": rng.randint(0, experts // 4)}
    if op in ("experts", "experts backward"):
        case.update(k=_spread(rng, 256, 2560, 128), n=_spread(rng, 256, 2048, 256), g=rng.choice((128, 128, -1)))
        if op == "experts":
            case["swiglu"] = rng.random() < 0.5
    else:
        case["k"] = _spread(rng, 64, 4096, 8)
    return case


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
    """Packed weights and their scales: entries of about 1 / sqrt(k)."""
    scales = (torch.rand((*lead, 1 if g == -1 else k // g, n), device=DEVICE, generator=gen) * 0.5 + 0.75) / (2.3 * math.sqrt(k))
    return _codes(gen, *lead, k // 16, 2 * n), scales.half()


def _choice(gen, case):
    """Each token's experts and their weights, some experts liked better than others; the last `away` of them are held elsewhere."""
    m, experts, top = case["m"], case["experts"], case["top"]
    scores = _normal(gen, m, experts) * 1.5 + _normal(gen, experts) * 0.4
    of = scores.argsort(dim=1, descending=True)[:, :top]
    weights = torch.softmax(torch.gather(scores, 1, of), dim=1)
    return torch.where(of >= experts - case["away"], -1, of).to(torch.int32), weights


def _sorted(of, experts):
    """(order, first, place) of a choice, as the operator gives them."""
    key = torch.where((of < 0) | (of >= experts), experts, of).reshape(-1).long()
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(len(order), device=DEVICE)
    counts = (key[:, None] == torch.arange(experts, device=DEVICE)).sum(0)
    first = torch.cat((torch.zeros_like(counts[:1]), counts.cumsum(0)))
    return order.to(torch.int32), first.to(torch.int32), place.reshape(of.shape).to(torch.int32)


def prepare(case, seed):
    gen, op = _generator(seed), case["op"]
    if op == "keep":
        m, n = case["m"], case["n"]
        gate_up = _normal(gen, m, 2 * n) * torch.exp(0.5 * _normal(gen, m, 1))
        return {"op": op, "gate_up": gate_up.to(torch.bfloat16), "dh": (_normal(gen, m, n) * 0.01).to(torch.bfloat16)}
    m, k, experts, top = case["m"], case["k"], case["experts"], case["top"]
    of, weights = _choice(gen, case)
    if op == "sort":
        return {"op": op, "x": _normal(gen, m, k).to(torch.bfloat16), "of": of, "experts": experts}
    order, first, place = _sorted(of, experts)
    state = {"op": op, "first": first, "place": place, "order": order, "experts": experts, "top": top}
    if op in ("combine", "combine backward"):
        state.update(rows=_normal(gen, m * top, k).to(torch.bfloat16), weights=weights)
    if op in ("sort backward", "combine backward"):
        state["dy"] = (_normal(gen, m * top if op == "sort backward" else m, k) * 0.01).to(torch.bfloat16)
    if op in ("experts", "experts backward"):
        n, g = case["n"], case["g"]
        state["counts"] = (first[1:] - first[:-1]).tolist()
        state["b"], state["s"] = _weight(gen, k, n, g, experts)
        state["g"] = g
        if op == "experts":
            state["swiglu"] = case["swiglu"]
            state["x"] = _normal(gen, m if case["swiglu"] else m * top, k).to(torch.bfloat16)
        else:
            state["dy"] = (_normal(gen, m * top, n) * 0.01).to(torch.bfloat16)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------

def run(s):
    name = s["op"].replace(" ", "_")
    return globals()["_own_" + name if own else "_" + name](s)


def _own_sort(s):
    from kiln_amd import marlin_gemm
    order, first, place = marlin_gemm.moe_sort(s["of"], s["experts"])
    return {"order": order, "first": first, "place": place, "rows": marlin_gemm.moe_gather(s["x"], first, place)}


def _own_sort_backward(s):
    from kiln_amd import marlin_gemm
    return marlin_gemm.moe_gather_backward(s["dy"], s["first"], s["place"])


def _own_combine(s):
    from kiln_amd import marlin_gemm
    return marlin_gemm.moe_combine(s["rows"], s["weights"], s["first"], s["place"])


def _own_combine_backward(s):
    from kiln_amd import marlin_gemm
    d_rows, d_weights = marlin_gemm.moe_combine_backward(s["dy"], s["rows"], s["weights"], s["first"], s["place"])
    return {"d_rows": d_rows, "d_weights": d_weights}


def _own_experts(s):
    from kiln_amd import marlin_gemm
    if s["swiglu"]:
        return marlin_gemm.marlin_w4a16_gemm_experts(s["x"], s["first"], s["b"], s["s"], s["g"], order=s["order"], top_k=s["top"], swiglu=True)
    return marlin_gemm.marlin_w4a16_gemm_experts(s["x"], s["first"], s["b"], s["s"], s["g"])


def _own_experts_backward(s):
    from kiln_amd import marlin_gemm
    return marlin_gemm.marlin_w4a16_gemm_experts_backward(s["dy"], s["first"], s["b"], s["s"], s["g"])


def _own_keep(s):
    from kiln_amd import marlin_gemm
    h, whole, exponents = marlin_gemm.swiglu_keep(s["gate_up"])
    d_gate_up, again = marlin_gemm.swiglu_keep_backward(s["dh"], whole, exponents, recompute=True)
    return {"h": h, "d_gate_up": d_gate_up, "again": again}


def _unpacked(b, scales):
    """A packed weight [k/16, 2n] and its scales as float32 [k, n]."""
    k, n = b.shape[0] * 16, b.shape[1] // 2
    groups = scales.shape[0]
    shifts = torch.tensor([4 * p for p in NIBBLE], dtype=torch.int32, device=b.device)
    words = b.reshape(n // 16, k // 128, 4, 16, 4, 1)                             # column tile, group, kq, column, t
    codes = ((words >> shifts) & 15).permute(1, 4, 2, 5, 0, 3)                    # group, t, kq, j, column tile, column
    w = (codes - 8).to(torch.float32).reshape(groups, k // groups, n)
    return (w * scales.reshape(n // 16, groups, 16).permute(1, 0, 2).reshape(groups, 1, n).to(torch.float32)).reshape(k, n)


def _sort(s):
    order, first, place = _sorted(s["of"], s["experts"])
    here = torch.arange(len(order), device=DEVICE) < first[-1]
    rows = torch.where(here[:, None], s["x"][order.long() // s["of"].shape[1]], torch.zeros_like(s["x"][:1]))
    return {"order": order, "first": first, "place": place, "rows": rows}


def _sort_backward(s):
    here = (s["place"] < s["first"][-1])[:, :, None]
    return torch.where(here, s["dy"][s["place"].long()].float(), 0).sum(1).to(torch.bfloat16)


def _combine(s):
    here = s["place"] < s["first"][-1]
    y = torch.zeros(s["place"].shape[0], s["rows"].shape[1], device=DEVICE)
    for j in range(s["place"].shape[1]):
        y += torch.where(here[:, j, None], s["rows"][s["place"][:, j].long()].float() * s["weights"][:, j, None], 0)
    return y.to(torch.bfloat16)


def _combine_backward(s):
    here = s["place"] < s["first"][-1]
    d_rows = torch.zeros_like(s["rows"])
    d_weights = torch.zeros_like(s["weights"])
    dy = s["dy"].float()
    for j in range(s["place"].shape[1]):
        at, ok = s["place"][:, j].long(), here[:, j, None]
        d_rows[at] = torch.where(ok, dy * s["weights"][:, j, None], 0).to(torch.bfloat16)
        d_weights[:, j] = torch.where(ok, dy * s["rows"][at].float(), 0).sum(1)
    return {"d_rows": d_rows, "d_weights": d_weights}


def _silu_times(gate_up):
    """silu(gate) * up of interleaved columns."""
    both = gate_up.reshape(gate_up.shape[0], -1, 2, 8)
    gate, up = both[:, :, 0].reshape(len(both), -1), both[:, :, 1].reshape(len(both), -1)
    return gate / (1 + torch.exp(-gate)) * up


def _experts(s):
    n = s["s"].shape[2] // (2 if s["swiglu"] else 1)
    y = torch.zeros(len(s["order"]), n, dtype=torch.bfloat16, device=DEVICE)
    at = 0
    for e, count in enumerate(s["counts"]):
        if count:
            rows = s["x"][s["order"][at:at + count].long() // s["top"]] if s["swiglu"] else s["x"][at:at + count]
            product = rows.float() @ _unpacked(s["b"][e], s["s"][e])
            y[at:at + count] = (_silu_times(product) if s["swiglu"] else product).to(torch.bfloat16)
        at += count
    return y


def _experts_backward(s):
    dx = torch.zeros(len(s["dy"]), s["b"].shape[1] * 16, dtype=torch.bfloat16, device=DEVICE)
    at = 0
    for e, count in enumerate(s["counts"]):
        if count:
            dx[at:at + count] = (s["dy"][at:at + count].float() @ _unpacked(s["b"][e], s["s"][e]).t()).to(torch.bfloat16)
        at += count
    return dx


def _in_eight_bits(gate_up):
    """What gate and up are kept as, and read back: float32 of the same shape."""
    m = gate_up.shape[0]
    blocks = gate_up.float().reshape(m, -1, 4, 2, 8).transpose(2, 3)              # 64 columns: [gate, up][4 x 8]
    most = blocks.abs().amax((3, 4), keepdim=True)
    byte = ((most.view(torch.int32) >> 23) & 255).clamp_min(1)
    whole = torch.round(torch.ldexp(blocks, 133 - byte)).clamp(-127, 127)
    return torch.ldexp(whole, byte - 133).transpose(2, 3).reshape(gate_up.shape)


def _keep(s):
    kept = _in_eight_bits(s["gate_up"]).reshape(s["dh"].shape[0], -1, 2, 8)
    gate, up, dh = kept[:, :, 0], kept[:, :, 1], s["dh"].float().reshape(kept[:, :, 0].shape)
    share = 1 / (1 + torch.exp(-gate))
    d_up, d_gate = dh * gate * share, dh * up * share * (1 + gate * (1 - share))
    return {"h": _silu_times(s["gate_up"].float()).to(torch.bfloat16),
            "d_gate_up": torch.stack((d_gate, d_up), 2).reshape(s["gate_up"].shape).to(torch.bfloat16),
            "again": (gate * share * up).reshape(s["dh"].shape).to(torch.bfloat16)}


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def work(case):
    m, op = case["m"], case["op"]
    if op == "keep":  # gate and up read, h and the 8 bits written; dh and the 8 bits read, the gradient and h again written
        n = case["n"]
        return {"bytes": m * n * (4 + 2 + 2.0625 + 2 + 2.0625 + 4 + 2), "flops": 30 * m * n}
    k, top, experts = case["k"], case["top"], case["experts"]
    pairs, share = m * top, (experts - case["away"]) / experts                    # of the pairs, those whose expert is here
    if op == "sort":
        return {"bytes": 2 * m * k + 2 * pairs * k + 12 * pairs + 4 * experts, "flops": 0}
    if op == "sort backward":
        return {"bytes": 2 * pairs * share * k + 2 * m * k + 4 * pairs, "flops": pairs * k}
    if op == "combine":
        return {"bytes": 2 * pairs * share * k + 2 * m * k + 8 * pairs, "flops": 2 * pairs * k}
    if op == "combine backward":
        return {"bytes": 2 * pairs * (1 + share) * k + 2 * m * k + 12 * pairs, "flops": 3 * pairs * k}
    n, g = case["n"], case["g"]
    used = (experts - case["away"]) * (1 - (1 - top / experts) ** m)
    weights = used * (k * n // 2 + (1 if g == -1 else k // g) * n * 2)
    if op == "experts":
        rows = m * k if case["swiglu"] else pairs * share * k
        return {"bytes": weights + 2 * rows + 2 * pairs * (n // 2 if case["swiglu"] else n), "flops": 2 * pairs * share * k * n}
    return {"bytes": weights + 2 * pairs * share * n + 2 * pairs * k, "flops": 2 * pairs * share * k * n}


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


def _exact_keep(s):
    m, columns = s["gate_up"].shape
    at = torch.arange(columns, device=DEVICE)
    gates, ups = at[at % 16 < 8], at[at % 16 >= 8]
    x = s["gate_up"].double()

    def kept(v):                                                                  # [m, n] of gate or of up
        blocks = v.reshape(m, -1, 32)
        unit = torch.exp2(torch.frexp(blocks.abs().amax(2, keepdim=True)).exponent.clamp_min(-125).double() - 7)
        return (torch.round(blocks / unit).clamp(-127, 127) * unit).reshape(v.shape)

    gate, up, dh = kept(x[:, gates]), kept(x[:, ups]), s["dh"].double()
    share = torch.sigmoid(gate)
    d = torch.empty_like(x)
    d[:, gates] = dh * up * (share + gate * share * (1 - share))
    d[:, ups] = dh * gate * share
    return {"h": x[:, gates] * torch.sigmoid(x[:, gates]) * x[:, ups], "d_gate_up": d, "again": gate * share * up}


def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    if op == "keep":
        return _exact_keep(s)
    if op == "sort":
        of, top = s["of"].reshape(-1).tolist(), s["of"].shape[1]
        pairs = [p for e in range(s["experts"]) for p in range(len(of)) if of[p] == e] if len(of) <= 4096 else \
            sorted((p for p in range(len(of)) if 0 <= of[p] < s["experts"]), key=lambda p: (of[p], p))
        rows = torch.zeros(len(of), s["x"].shape[1], dtype=torch.float64, device=DEVICE)
        rows[:len(pairs)] = s["x"][torch.tensor(pairs, dtype=torch.int64, device=DEVICE) // top].double()
        return {"order": None, "first": None, "place": None, "rows": rows}
    m, top = s["place"].shape
    order, placed = s["order"].long(), int(s["first"][-1])
    pairs = order[:placed]                                                        # the pairs that have an expert, by position
    if op == "sort backward":
        return torch.zeros(m, s["dy"].shape[1], dtype=torch.float64, device=DEVICE).index_add_(0, pairs // top, s["dy"][:placed].double())
    if op == "combine":
        weighted = s["rows"][:placed].double() * s["weights"].reshape(-1)[pairs].double()[:, None]
        return torch.zeros(m, s["rows"].shape[1], dtype=torch.float64, device=DEVICE).index_add_(0, pairs // top, weighted)
    if op == "combine backward":
        dy = s["dy"].double()[pairs // top]
        d_rows = torch.zeros(m * top, dy.shape[1], dtype=torch.float64, device=DEVICE)
        d_rows[:placed] = dy * s["weights"].reshape(-1)[pairs].double()[:, None]
        d_weights = torch.zeros(m * top, dtype=torch.float64, device=DEVICE)
        d_weights[pairs] = (dy * s["rows"][:placed].double()).sum(1)
        return {"d_rows": d_rows, "d_weights": d_weights.reshape(m, top)}
    bounds = s["first"].tolist()
    n = s["s"].shape[2]
    swiglu = op == "experts" and s["swiglu"]
    out = torch.zeros(m * top, s["b"].shape[1] * 16 if op == "experts backward" else n // 2 if swiglu else n, dtype=torch.float64, device=DEVICE)
    gates = [i for i in range(n) if i % 16 < 8]
    ups = [i + 8 for i in gates]
    for e in range(s["experts"]):
        i, j = bounds[e], bounds[e + 1]
        if i == j:
            continue
        w = _exact_weight(s["b"][e], s["s"][e])
        if op == "experts backward":
            out[i:j] = s["dy"][i:j].double() @ w.t()
            continue
        y = (s["x"][order[i:j] // top] if swiglu else s["x"][i:j]).double() @ w
        out[i:j] = y[:, gates] * torch.sigmoid(y[:, gates]) * y[:, ups] if swiglu else y
    return out

"""Operators on rows that each name the weights they use, timed as a serving
step calls them, with a plain form of each.

  route     router logits [tokens, experts] -> each token's top_k experts, their
            softmax weights, and the rows grouped by expert (order, slots,
            offsets).
  combine   the experts' outputs back to tokens: sum_j weight[t, j] *
            h[slots[t, j]], plus an optional 16-bit base row.
  experts   the quantized product of each group's rows with its own weights:
            INT8 / FP8 codes, per-channel scales or K groups of 128, the rows
            gathered through `order`, the results in slot order or scattered to
            the rows they came from.
  adapters  y[m] = base[m] + scale[a] * B[a] (A[a] x[m]) for the rows of adapter a:
            low-rank adapters of many requests beside one shared projection.
            Rows of no adapter keep y as it was.

Sizes: the widths are the decoder projections' (2048, 4096, 6144, 12288) and
1024 for an expert's intermediate; row counts are decode batches (1-64), prompts
(187, 431, 1000) and prefill (4096).
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------- cases
def _route(tokens, experts, top_k, dtype, normalize, masked=0):
    return {"kind": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype,
            "normalize": normalize, "masked": masked}


def _combine(tokens, top_k, N, dtype, base, masked=0):
    return {"kind": "combine", "tokens": tokens, "top_k": top_k, "N": N, "dtype": dtype, "base": base,
            "masked": masked}


def _experts(tokens, top_k, experts, N, K, mode, gather, scatter=False, dtype="bf16", masked=0):
    return {"kind": "experts", "tokens": tokens, "top_k": top_k, "experts": experts, "N": N, "K": K,
            "mode": mode, "gather": gather, "scatter": scatter, "dtype": dtype, "masked": masked}


def _adapters(rows, adapters, rank, N, K, dtype, ragged=False, absent=0.0, ids=False, pad=0):
    return {"kind": "adapters", "rows": rows, "adapters": adapters, "rank": rank, "N": N, "K": K,
            "dtype": dtype, "ragged": ragged, "absent": absent, "ids": ids, "pad": pad}


def listed():
    return [
        # A decode step's router: 16 requests, fp32 logits; latency is all of it.
        dict(_route(16, 64, 6, "f32", True), name="route_decode"),
        # A prefill's router on 16-bit logits (ties are common), the last 63 rows padding.
        dict(_route(8191, 128, 8, "bf16", False, masked=63), name="route_prefill"),
        # The same step's return of the experts' rows to their tokens.
        dict(_combine(16, 6, 2048, "bf16", False), name="combine_decode"),
        # A prefill's return, onto the shared expert's output.
        dict(_combine(4096, 8, 2048, "bf16", True, masked=31), name="combine_prefill"),
        # One request's token: eight experts' gate and up weights are streamed once.
        dict(_experts(1, 8, 64, 2048, 2048, "int8", True), name="experts_token_int8"),
        # A decode batch's down product: nearly every expert has a few rows.
        dict(_experts(32, 6, 64, 2048, 1024, "fp8", False), name="experts_decode_fp8"),
        # Requests at different codebooks, each row through its codebook's own head
        # (2051 entries and padding), the results back in request order.
        dict(_experts(187, 1, 31, 2064, 2048, "group_int8", True, scatter=True),
             name="heads_batch_group_int8"),
        # A prompt's down product with K groups, the last tokens padding.
        dict(_experts(1000, 8, 64, 2048, 1024, "group_fp8", False, masked=40),
             name="experts_prompt_group_fp8"),
        # A prefill's gate and up product: compute bound.
        dict(_experts(4096, 4, 32, 4096, 2048, "int8", True), name="experts_prefill_int8"),
        # One request with its own voice.
        dict(_adapters(1, 8, 16, 4096, 2048, "bf16"), name="adapters_token"),
        # A decode batch of many voices of several ranks, some rows with none, grouped in
        # the step; x is a slice of wider rows.
        dict(_adapters(57, 16, 32, 12288, 2048, "bf16", ragged=True, absent=0.2, ids=True, pad=64),
             name="adapters_decode"),
        # A prefill of a few requests, a large rank.
        dict(_adapters(4096, 6, 64, 2048, 6144, "f16"), name="adapters_prefill"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    return min(hi, max(lo, (_log(rng, lo, hi) + 8) // 16 * 16))


def draw(rng):
    kind = rng.choice(["route", "combine", "experts", "experts", "adapters"])
    if kind == "route":
        tokens, experts = _log(rng, 1, 8000), _log(rng, 4, 128)
        return _route(tokens, experts, rng.randint(1, min(8, experts)),
                      rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.5,
                      rng.randint(0, tokens // 8))
    if kind == "combine":
        tokens, N = _log(rng, 1, 4000), _width(rng, 256, 4096)
        top_k = max(1, min(rng.randint(1, 8), 4096 * 8 * 2048 // (tokens * N)))
        return _combine(tokens, top_k, N, rng.choice(["bf16", "f16"]), rng.random() < 0.5,
                        rng.randint(0, tokens // 8))
    if kind == "experts":
        while True:
            tokens, experts = _log(rng, 1, 4096), _log(rng, 2, 64)
            top_k = rng.randint(1, min(8, experts))
            N, K = _width(rng, 256, 4096), _width(rng, 256, 4096)
            if tokens * top_k * N * K <= 4096 * 4 * 4096 * 2048:
                break
        gather = rng.random() < 0.6
        return _experts(tokens, top_k, experts, N, K,
                        rng.choice(["int8", "fp8", "group_int8", "group_fp8"]), gather,
                        gather and rng.random() < 0.3, rng.choice(["bf16", "f16"]),
                        rng.randint(0, tokens // 8))
    while True:
        rows, adapters = _log(rng, 1, 4096), _log(rng, 1, 32)
        rank = rng.choice([4, 8, 12, 16, 24, 32, 64, 128])
        N, K = _width(rng, 256, 12288), _width(rng, 256, 6144)
        if rows * (N + K) * 2 <= 4096 * 8192 * 2 and adapters * rank * (N + K) <= 1 << 26:
            break
    return _adapters(rows, adapters, rank, N, K, rng.choice(["bf16", "f16"]), rng.random() < 0.5,
                     rng.choice([0.0, 0.2]), rng.random() < 0.5, rng.choice([0, 0, 8, 9]))


# ---------------------------------------------------------------- inputs
def _rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _group(ids, groups):
    """order, slots, offsets of flat ids: a stable sort; ids outside [0, groups) have no slot."""
    count = ids.numel()
    key = torch.where((ids >= 0) & (ids < groups), ids, torch.full_like(ids, groups)).long()
    order = torch.sort(key, stable=True)[1]
    have = (key[:, None] == torch.arange(groups + 1, device=ids.device)[None, :]).sum(0)
    offsets = torch.cat([have.new_zeros(1), torch.cumsum(have[:groups], 0)])
    place = torch.arange(count, device=ids.device)
    used = place < offsets[groups]
    slots = torch.empty_like(place)
    slots[order] = torch.where(used, place, torch.full_like(place, -1))
    order = torch.where(used, order, torch.full_like(order, -1))
    return order.int(), slots.int(), offsets.int()


def _choices(g, tokens, experts, top_k, masked):
    """Router choices [tokens, top_k] of an uneven popularity; padding rows choose none."""
    logits = _randn(g, tokens, experts) + 0.5 * _randn(g, experts)
    ids = torch.topk(logits, top_k, dim=1)[1].int()
    ids[tokens - masked:] = -1
    return ids


def _codes(g, rows, K, mode, spread):
    """Codes (uint8 [rows, K]) and scales ([rows] or [groups, rows]) of normal values."""
    fmt, group = ("fp8" if "fp8" in mode else "int8"), (128 if "group" in mode else 0)
    v = _randn(g, rows, K)
    if fmt == "int8":
        q = torch.round(v * 32).clamp_(-127, 127).to(torch.int8).view(torch.uint8)
        unit = spread / 32
    else:
        q = (v * 100).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        unit = spread / 100
    shape = ((K + group - 1) // group, rows) if group else (rows,)
    return q, unit * (0.75 + 0.5 * torch.rand(*shape, generator=g, device="cuda"))


def prepare(case, seed):
    g = _rng(seed)
    kind, state = case["kind"], {"case": dict(case)}
    if kind == "route":
        t, e = case["tokens"], case["experts"]
        logits = (2 * _randn(g, t, e) + _randn(g, e)).to(DTYPES[case["dtype"]])
        # Some experts are switched off for some tokens; padding rows have none left.
        logits[torch.rand(t, e, generator=g, device="cuda") < 0.02] = float("-inf")
        logits[t - case["masked"]:] = float("-inf")
        state["logits"] = logits
    elif kind == "combine":
        t, k, N, dt = case["tokens"], case["top_k"], case["N"], DTYPES[case["dtype"]]
        experts = max(16, 2 * k)
        ids = _choices(g, t, experts, k, case["masked"])
        state["order"], state["slots"], state["offsets"] = _group(ids.flatten(), experts)
        state["slots"] = state["slots"].view(t, k)
        state["weights"] = torch.softmax(_randn(g, t, k), 1)
        state["h"] = _randn(g, t * k, N).to(dt)
        state["base"] = _randn(g, t, N).to(dt) if case["base"] else None
    elif kind == "experts":
        t, k, e, N, K = (case[n] for n in ("tokens", "top_k", "experts", "N", "K"))
        ids = _choices(g, t, e, k, case["masked"])
        state["order"], state["slots"], state["offsets"] = _group(ids.flatten(), e)
        rows = t if case["gather"] else t * k
        state["x"], state["sx"] = _codes(g, rows, K, case["mode"], 1.0)
        w = [_codes(g, N, K, case["mode"], 0.02) for _ in range(e)]
        state["w"], state["sw"] = torch.stack([a for a, _ in w]), torch.stack([b for _, b in w])
        state["y"] = torch.zeros(t * k, N, dtype=DTYPES[case["dtype"]], device="cuda")
    else:
        rows, n, r, N, K = (case[m] for m in ("rows", "adapters", "rank", "N", "K"))
        dt, pad = DTYPES[case["dtype"]], case["pad"]
        # Requests are runs of rows with one adapter; in decode every row is its own.
        run = 1 if rows <= 64 else max(1, rows // (2 * n))
        requests = (rows + run - 1) // run
        ids = torch.randint(0, n, (requests,), generator=g, device="cuda")
        none = torch.rand(requests, generator=g, device="cuda") < case["absent"]
        ids = torch.where(none, torch.full_like(ids, -1), ids).repeat_interleave(run)[:rows].int()
        state["ids"] = ids.contiguous()
        state["order"], _, state["offsets"] = _group(ids, n)
        state["x"] = _randn(g, rows, K + pad).to(dt)[:, pad:]
        state["a"] = (_randn(g, n, r, K) / math.sqrt(K)).to(dt)
        state["b"] = (_randn(g, n, N, r) / math.sqrt(r)).to(dt)
        state["scales"] = 0.5 + torch.rand(n, generator=g, device="cuda")
        state["ranks"] = None
        if case["ragged"]:
            pick = torch.randint(0, 3, (n,), generator=g, device="cuda")
            state["ranks"] = torch.clamp(r >> pick, min=1).int()
        state["base"] = _randn(g, rows, N).to(dt)
        state["y"] = state["base"].clone()
    return state


# ---------------------------------------------------------------- one pass
def _values(codes, mode):
    return codes.view(torch.float8_e4m3fn if "fp8" in mode else torch.int8).float()


def _dequantized(codes, scales, mode):
    v = _values(codes, mode)
    if "group" in mode:
        return v * scales.repeat_interleave(128, 0)[:v.shape[1]].t()
    return v * scales[:, None]


def _run_route(s):
    c = s["case"]
    if own:
        from breeze_tts_cpp_amd import qlinear
        ids, weights, order, slots, offsets = qlinear.route(s["logits"], c["top_k"],
                                                            normalize=c["normalize"])
    else:
        v = s["logits"].float()
        top, ids = torch.sort(v, dim=1, descending=True, stable=True)
        top, ids = top[:, :c["top_k"]], ids[:, :c["top_k"]]
        there = top > float("-inf")
        peak = torch.where(there[:, :1], top[:, :1], torch.zeros_like(top[:, :1]))
        p = torch.exp(top - peak)
        total = p if c["normalize"] else torch.exp(v - peak)
        weights = torch.where(there, p / total.sum(1, keepdim=True), torch.zeros_like(p))
        ids = torch.where(there, ids, torch.full_like(ids, -1)).int()
        order, slots, offsets = _group(ids.flatten(), c["experts"])
        slots = slots.view_as(ids)
    return {"ids": ids, "weights": weights, "order": order, "slots": slots, "offsets": offsets}


def _run_combine(s):
    if own:
        from breeze_tts_cpp_amd import qlinear
        return qlinear.combine(s["h"], s["slots"], s["weights"], base=s["base"])
    rows = s["h"][s["slots"].clamp(min=0).long()].float()
    there = (s["slots"] >= 0)[:, :, None]
    y = (torch.where(there, rows, torch.zeros_like(rows)) * s["weights"][:, :, None]).sum(1)
    if s["base"] is not None:
        y = y + s["base"].float()
    return y.to(s["h"].dtype)


def _run_experts(s):
    c = s["case"]
    mode, y = c["mode"], s["y"]
    if own:
        from breeze_tts_cpp_amd import qlinear
        return qlinear.expert_gemm(s["x"], s["sx"], s["w"], s["sw"],
                                   qlinear.FP8 if "fp8" in mode else qlinear.I8, s["offsets"],
                                   order=s["order"] if c["gather"] else None,
                                   divisor=c["top_k"], scatter=c["scatter"],
                                   group=128 if "group" in mode else 0, out=y)
    x = _dequantized(s["x"], s["sx"], mode)
    ends = s["offsets"].tolist()
    for e in range(c["experts"]):
        begin, end = ends[e], ends[e + 1]
        if begin == end:
            continue
        rows = s["order"][begin:end].long()
        part = x[rows // c["top_k"]] if c["gather"] else x[begin:end]
        out = torch.matmul(part, _dequantized(s["w"][e], s["sw"][e], mode).t()).to(y.dtype)
        if c["scatter"]:
            y[rows] = out
        else:
            y[begin:end] = out
    return y


def _run_adapters(s):
    c = s["case"]
    n = c["adapters"]
    if own:
        from breeze_tts_cpp_amd import qlinear
        order, offsets = s["order"], s["offsets"]
        if c["ids"]:
            order, _, offsets = qlinear.group_rows(s["ids"], n)
        return qlinear.adapter_add(s["x"], order, offsets, s["a"], s["b"], s["y"], base=s["base"],
                                   ranks=s["ranks"], scales=s["scales"])
    order, offsets = s["order"], s["offsets"]
    if c["ids"]:
        order, _, offsets = _group(s["ids"], n)
    y, ends = s["y"], offsets.tolist()
    ranks = [c["rank"]] * n if s["ranks"] is None else s["ranks"].tolist()
    for i in range(n):
        if ends[i] == ends[i + 1]:
            continue
        rows, r = order[ends[i]:ends[i + 1]].long(), ranks[i]
        t = torch.matmul(s["x"][rows].float(), s["a"][i, :r].float().t())
        delta = torch.matmul(t, s["b"][i, :, :r].float().t()) * s["scales"][i]
        y[rows] = (s["base"][rows].float() + delta).to(y.dtype)
    return y


def run(state):
    return {"route": _run_route, "combine": _run_combine, "experts": _run_experts,
            "adapters": _run_adapters}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- work
def _hit(groups, rows_each, draws):
    """Groups that `draws` independent picks of `rows_each` distinct ones reach, on average."""
    return groups * (1 - (1 - rows_each / groups) ** draws)


def work(case):
    kind = case["kind"]
    if kind == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": t * e * size + t * k * 16 + (e + 1) * 4, "flops": t * e * 2}
    if kind == "combine":
        t, k, N = case["tokens"], case["top_k"], case["N"]
        live = t - case["masked"]
        return {"bytes": live * k * N * 2 + t * N * 2 * (2 if case["base"] else 1) + t * k * 8,
                "flops": 2 * live * k * N}
    if kind == "experts":
        t, k, e, N, K = (case[n] for n in ("tokens", "top_k", "experts", "N", "K"))
        live = t - case["masked"]
        scales = (K + 127) // 128 if "group" in case["mode"] else 1
        rows = live if case["gather"] else live * k
        return {"bytes": int(_hit(e, k, live) * N * (K + 4 * scales)) + rows * (K + 4 * scales)
                + live * k * N * 2 + live * k * 4 + e * 4,
                "flops": 2 * live * k * N * K}
    rows, n, r, N, K = (case[m] for m in ("rows", "adapters", "rank", "N", "K"))
    live = int(rows * (1 - case["absent"]))
    mean = r * 7 / 12 if case["ragged"] else r
    requests = rows if rows <= 64 else 2 * n
    return {"bytes": int(_hit(n, 1, requests * (1 - case["absent"])) * mean * (N + K) * 2)
            + live * (K + 2 * N) * 2 + rows * 4,
            "flops": int(2 * live * mean * (N + K))}


# ---------------------------------------------------------------- in 64 bits
def _exact_codes(codes, scales, mode):
    """Codes times scales in float64, K by blocks of 128."""
    kind = torch.float8_e4m3fn if "fp8" in mode else torch.int8
    v = codes.view(kind).to(torch.float32).double()
    if "group" not in mode:
        return v * scales.double().unsqueeze(1)
    for b in range(scales.shape[0]):
        v[:, b * 128:(b + 1) * 128] *= scales[b].double().unsqueeze(1)
    return v


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        # Experts by repeated arg max, the first of equals; only the weights are computed numbers.
        v = s["logits"].double()
        left, tokens, k = v.clone(), case["tokens"], case["top_k"]
        weights = torch.zeros(tokens, k, dtype=torch.float64, device="cuda")
        best = left.max(1)[0]
        for j in range(k):
            top = left.max(1)[0]
            at = (left == top[:, None]).int().argmax(1)
            live = top > -math.inf
            weights[live, j] = torch.exp(top[live] - best[live])
            left[torch.arange(tokens, device="cuda"), at] = -math.inf
        below = weights.sum(1)
        if not case["normalize"]:
            below = torch.exp(v - torch.where(best > -math.inf, best, 0.0)[:, None]).sum(1)
        weights = weights / torch.where(below > 0, below, 1.0)[:, None]
        return {"ids": None, "weights": weights, "order": None, "slots": None, "offsets": None}
    if kind == "combine":
        out = torch.zeros(case["tokens"], case["N"], dtype=torch.float64, device="cuda")
        for j in range(case["top_k"]):
            at = s["slots"][:, j]
            live = at >= 0
            out[live] += s["weights"][live, j].double()[:, None] * s["h"][at[live].long()].double()
        return out if s["base"] is None else out + s["base"].double()
    if kind == "experts":
        out = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
        x = _exact_codes(s["x"], s["sx"], case["mode"])
        # Each slot's expert from the offsets, then the slots of every expert.
        place = torch.arange(out.shape[0], device="cuda")
        of = (place[:, None] >= s["offsets"][None, 1:].long()).sum(1)
        for e in range(case["experts"]):
            mine = place[of == e]
            if not mine.numel():
                continue
            flat = s["order"][mine].long()
            source = torch.div(flat, case["top_k"], rounding_mode="floor") if case["gather"] else mine
            out[flat if case["scatter"] else mine] = x[source] @ _exact_codes(s["w"][e], s["sw"][e], case["mode"]).t().contiguous()
        return out
    out = s["base"].double()
    for i in range(case["adapters"]):
        rows = torch.nonzero(s["ids"] == i).flatten()
        r = case["rank"] if s["ranks"] is None else int(s["ranks"][i])
        a, b = s["a"][i, :r].double(), s["b"][i, :, :r].double()
        t = s["x"][rows].double() @ a.t().contiguous()
        out[rows] += float(s["scales"][i]) * (t @ b.t().contiguous())
    return out

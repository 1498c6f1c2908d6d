"""The operators around a sparse layer whose experts are held in 4 bits, as a program that serves or tunes
such a layer calls them: the norm before it, the tokens sorted by expert and back, and the experts' products.

``listed()`` names the measured cases and ``draw()`` makes more of the same ranges.  ``run()`` is one pass:
elementary torch operations where ``own`` is false, the framework's entry points where it is true.  ``exact()``
is the same pass in 64 bits, straight from the definitions.
"""
import math
import random

import torch

own = False

EPS = 1e-6
QBLOCK = 128  # elements of a row that share one scale in 8 bits
FP8_MAX = 448.0

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}


def ceil_div(a, b):
    return -(-a // b)


# ---- the cases ------------------------------------------------------------------------------------------


def norm_case(T, H, dtype, out8, residual=True):
    """Residual added, RMS norm of the sum, the sum kept; out8: the norm leaves in e4m3 with scales."""
    return {"op": "norm", "T": T, "H": H, "dtype": dtype, "out8": out8, "residual": residual}


def sort_case(T, H, dtype, K=8, E=256, absent=0.0, grad=False):
    """T tokens with K routes each, sorted by expert; absent: share of routes to experts held elsewhere."""
    return {"op": "sort", "T": T, "H": H, "dtype": dtype, "K": K, "E": E, "absent": absent, "grad": grad}


def unsort_case(T, H, dtype, out="bf16", K=8, E=256, absent=0.0, residual=True, grad=False):
    """The experts' rows back to their tokens, weighted and summed."""
    return {"op": "unsort", "T": T, "H": H, "dtype": dtype, "out": out, "K": K, "E": E, "absent": absent,
            "residual": residual, "grad": grad}


def int4_case(R, E, N, K, dtype, group=128, zeros=False, swiglu=False, skew=0.5, tail=0):
    """R rows sorted by expert times E weights [N, K] of 4 bits; tail: rows behind the last expert's."""
    return {"op": "int4", "R": R, "E": E, "N": N, "K": K, "dtype": dtype, "group": group, "zeros": zeros,
            "swiglu": swiglu, "skew": skew, "tail": tail}


def listed():
    return [
        # one new token: the norm's latency
        dict(norm_case(1, 7168, "bf16", True), name="norm to 8 bits, one token"),
        # a prefill chunk through the norm that feeds 8-bit products
        dict(norm_case(4096, 7168, "bf16", True), name="norm to 8 bits, chunk"),
        # a ragged batch of a width that no vector load divides
        dict(norm_case(333, 5001, "fp16", False), name="norm, odd width"),
        # a decode step's dispatch
        dict(sort_case(64, 7168, "bf16"), name="sort, decode batch"),
        # a prefill chunk's dispatch in 8 bits, one route in eight held on another device
        dict(sort_case(4096, 7168, "fp8", absent=0.125), name="sort 8 bits, chunk"),
        # a tuning step's dispatch, with the gradient of the tokens
        dict(sort_case(2048, 7168, "bf16", grad=True), name="sort and gradient"),
        # a decode step's combine
        dict(unsort_case(64, 7168, "bf16"), name="unsort, decode batch"),
        # a tuning step's combine, with the gradients of rows and weights
        dict(unsort_case(4096, 7168, "bf16", residual=False, grad=True), name="unsort and gradients"),
        # one token through one expert's up and gate
        dict(int4_case(1, 1, 4096, 7168, "bf16", swiglu=True), name="int4 up/gate, one row"),
        # a node's batch through 32 experts' down products, asymmetric weights
        dict(int4_case(254, 32, 7168, 2048, "fp16", group=64, zeros=True), name="int4 down, 32 experts"),
        # a decode layer's up and gate on one rank of four
        dict(int4_case(512, 64, 4096, 7168, "bf16", swiglu=True), name="int4 up/gate, 64 experts"),
        # few experts with many rows each, rows as the 8-bit norm leaves them
        dict(int4_case(200, 8, 4096, 7168, "fp8", tail=9), name="int4 of 8-bit rows"),
    ]


def log_int(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.25 / hi)))))


def width(rng, lo, hi):
    """A row width: half of them multiples of 128, a quarter multiples of 8, the others as they fall."""
    h = log_int(rng, lo, hi)
    kind = rng.random()
    return max(128, h // 128 * 128) if kind < 0.5 else max(8, h // 8 * 8) if kind < 0.75 else h


def draw(rng):
    op = rng.choice(("norm", "sort", "unsort", "int4", "int4"))
    if op == "norm":
        H = width(rng, 64, 16384)
        out8 = rng.random() < 0.6
        return norm_case(log_int(rng, 1, 4096 * 7168 // H), H, rng.choice(("bf16", "bf16", "fp16", "fp32")), out8,
                         rng.random() < 0.8 or not out8)
    if op in ("sort", "unsort"):
        H, K = width(rng, 64, 8192), rng.choice((1, 2, 4, 6, 8, 8))
        E = rng.choice((4, 16, 60, 64, 160, 256))
        E = max(E, K)
        T = log_int(rng, 1, 2048 * 8 * 7168 // (H * K))
        absent, grad = rng.choice((0.0, 0.0, 0.25, 0.75)), rng.random() < 0.4
        if op == "sort":
            dtype = rng.choice(("bf16", "bf16", "fp16", "fp32", "fp8"))
            return sort_case(T, H, dtype, K, E, absent, grad and dtype != "fp8")
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        return unsort_case(T, H, dtype, rng.choice((dtype, "fp32")), K, E, absent, rng.random() < 0.5, grad)
    group = rng.choice((32, 64, 128, 128))
    swiglu = rng.random() < 0.4
    K = ceil_div(log_int(rng, 256, 8192), group) * group
    N = log_int(rng, 256, 8192)
    N = ceil_div(N, 32) * 32 if swiglu else N
    E = log_int(rng, 1, max(1, min(128, 32 * 4096 * 7168 // (N * K))))
    return int4_case(log_int(rng, 1, 512), E, N, K, rng.choice(("bf16", "bf16", "fp16", "fp8")), group,
                     rng.random() < 0.4, swiglu, rng.choice((0.0, 0.5, 1.5)), rng.choice((0, 0, 3)))


def expert_rows(case):
    """Rows of each expert, from the case alone: log-normal shares, whole numbers by largest remainder."""
    E, R = case["E"], case["R"]
    r = random.Random("%d %d %s" % (E, R, case["skew"]))
    share = [math.exp(case["skew"] * r.gauss(0, 1)) for _ in range(E)]
    total = sum(share)
    want = [R * s / total for s in share]
    got = [int(w) for w in want]
    rest = sorted(range(E), key=lambda e: (got[e] - want[e], e))
    for e in rest[:R - sum(got)]:
        got[e] += 1
    return got


def work(case):
    op = case["op"]
    if op == "norm":
        T, H, s = case["T"], case["H"], SIZE[case["dtype"]]
        b = T * H * s * (3 if case["residual"] else 1) + 4 * H
        b += T * (H + 4 * ceil_div(H, QBLOCK)) if case["out8"] else T * H * s
        return {"bytes": b, "flops": 5 * T * H}
    if op in ("sort", "unsort"):
        T, H, K, s = case["T"], case["H"], case["K"], SIZE[case["dtype"]]
        here = T * K * (1.0 - case["absent"])
        if op == "sort":
            b = T * K * (4 + 8) + T * H * s + T * K * H * s
            b += (T + T * K) * 4 * ceil_div(H, QBLOCK) if case["dtype"] == "fp8" else 0
            b += here * H * s + T * H * s if case["grad"] else 0
            return {"bytes": b, "flops": here * H if case["grad"] else 0}
        o = SIZE[case["out"]]
        b = T * K * 8 + here * H * s + T * H * o * (2 if case["residual"] else 1)
        if case["grad"]:  # rows and the result's gradient are read again, the rows' gradient is written whole
            b += here * H * s + T * H * o + T * K * H * s + T * K * 8
        return {"bytes": b, "flops": here * H * (5 if case["grad"] else 2)}
    N, K, s = case["N"], case["K"], SIZE[case["dtype"]]
    rows = expert_rows(case)
    used = sum(n > 0 for n in rows)
    per = N * K // 2 + N * (K // case["group"]) * 2 + (N * (K // case["group"]) // 2 if case["zeros"] else 0)
    out = (N // 2 if case["swiglu"] else N) * (2 if case["dtype"] != "fp32" else 4)
    b = used * per + case["R"] * K * s + (case["R"] + case["tail"]) * out + 4 * (case["E"] + 1)
    b += case["R"] * ceil_div(K, QBLOCK) * 4 if case["dtype"] == "fp8" else 0
    return {"bytes": b, "flops": 2 * case["R"] * N * K}


# ---- inputs ---------------------------------------------------------------------------------------------


def activations(g, rows, cols, dtype):
    """Normalised rows, each token at its own magnitude, as a hidden state has them."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    x *= torch.exp(0.3 * torch.randn(rows, 1, generator=g, device="cuda"))
    return x.to(DTYPES[dtype])


def rows8(g, rows, cols):
    """Rows in e4m3 with one scale for 128 elements."""
    q = (torch.randn(rows, cols, generator=g, device="cuda") * 120).clamp_(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    scale = torch.exp(0.3 * torch.randn(rows, ceil_div(cols, QBLOCK), generator=g, device="cuda")) / 120
    return q, scale


def routes(g, T, K, E, absent):
    """K different experts for each token with weights that sum to 2.5; -1 where the expert is held elsewhere."""
    pref = torch.randn(T, E, generator=g, device="cuda") + torch.linspace(0.0, 1.0, E, device="cuda")
    idx = torch.topk(pref, K, dim=1).indices.to(torch.int32)
    weight = torch.rand(T, K, generator=g, device="cuda") + 0.1
    weight = weight * (2.5 / weight.sum(dim=1, keepdim=True))
    if absent:
        idx = torch.where(torch.rand(T, K, generator=g, device="cuda") < absent, torch.full_like(idx, -1), idx)
    return idx, weight


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, s = case["op"], {"case": case}
    if op == "norm":
        s["x"] = activations(g, case["T"], case["H"], case["dtype"])
        s["residual"] = activations(g, case["T"], case["H"], case["dtype"]) if case["residual"] else None
        s["weight"] = 1.0 + 0.1 * torch.randn(case["H"], generator=g, device="cuda")
    elif op == "sort":
        s["idx"], _ = routes(g, case["T"], case["K"], case["E"], case["absent"])
        if case["dtype"] == "fp8":
            s["x"], s["scale"] = rows8(g, case["T"], case["H"])
        else:
            s["x"] = activations(g, case["T"], case["H"], case["dtype"])
        if case["grad"]:
            s["x"].requires_grad_()
            s["grad"] = activations(g, case["T"] * case["K"], case["H"], case["dtype"])
    elif op == "unsort":
        idx, s["weight"] = routes(g, case["T"], case["K"], case["E"], case["absent"])
        s["row_of"], s["route_of"], s["offsets"] = plain_order(idx, case["E"])
        s["rows"] = activations(g, case["T"] * case["K"], case["H"], case["dtype"])
        s["residual"] = activations(g, case["T"], case["H"], case["out"]) if case["residual"] else None
        if case["grad"]:
            s["rows"].requires_grad_()
            s["weight"].requires_grad_()
            s["grad"] = activations(g, case["T"], case["H"], case["out"])
    else:
        E, N, K, G = case["E"], case["N"], case["K"], case["K"] // case["group"]
        R = case["R"] + case["tail"]
        # as a quantised checkpoint has them: two values a byte, the lower k in the lower half
        q = (torch.randn(E, N, K // 2, 2, generator=g, device="cuda", dtype=torch.float16) * 2.6 + 8).round_()
        q = q.clamp_(0, 15).to(torch.uint8)
        s["q"] = q[..., 0] | (q[..., 1] << 4)
        del q
        s["wscale"] = (torch.exp(0.25 * torch.randn(E, N, G, generator=g, device="cuda")) * 0.0075).to(torch.float16)
        s["zero"] = None
        if case["zeros"]:
            s["zero"] = (torch.randn(E, N, G, generator=g, device="cuda") + 7.5).round_().clamp_(0, 15).to(torch.uint8)
        count = expert_rows(case)
        random.Random(int(seed)).shuffle(count)
        s["most"] = max(count)
        s["offsets"] = torch.tensor([0] + count, device="cuda").cumsum(0).to(torch.int32)
        if case["dtype"] == "fp8":
            s["x"], s["scale"] = rows8(g, R, K)
        else:
            s["x"], s["scale"] = activations(g, R, K, case["dtype"]), None
        if own:
            from constellation_b200.int4 import Int4Weight

            s["w"] = Int4Weight(s["q"], s["wscale"], s["zero"], swiglu=case["swiglu"])
            del s["q"], s["wscale"], s["zero"]
    return s


# ---- the plain forms ------------------------------------------------------------------------------------


def plain_norm(s):
    case, h = s["case"], s["x"].float()
    if case["residual"]:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * s["weight"]
    kept = h.to(s["x"].dtype) if case["residual"] else None
    if not case["out8"]:
        return {"out": y.to(s["x"].dtype), "sum": kept}
    T, H = y.shape
    B = ceil_div(H, QBLOCK)
    y = torch.nn.functional.pad(y, (0, B * QBLOCK - H)).view(T, B, QBLOCK)
    most = y.abs().amax(dim=2, keepdim=True)
    scale = torch.where(most > 0, most / FP8_MAX, torch.ones_like(most))
    q = (y / scale).clamp(-FP8_MAX, FP8_MAX).view(T, B * QBLOCK)[:, :H].to(torch.float8_e4m3fn)
    return {"out": q, "scale": scale.view(T, B), "sum": kept}


def plain_order(idx, E):
    """The row of each route in the order (expert, token, k), the route of each row, the experts' first rows."""
    flat = idx.reshape(-1).long()
    here = (flat >= 0) & (flat < E)
    key = torch.where(here, flat, torch.full_like(flat, E))
    route = torch.sort(key, stable=True).indices
    row = torch.empty_like(route)
    row[route] = torch.arange(route.numel(), device=route.device)
    offsets = torch.searchsorted(key[route], torch.arange(E + 1, device=key.device)).to(torch.int32)
    absent = torch.full_like(row, -1)
    return (torch.where(here, row, absent).to(torch.int32).view(idx.shape),
            torch.where(here[route], route, absent).to(torch.int32), offsets)


def plain_sort(s):
    case, x = s["case"], s["x"].detach()
    row_of, route_of, offsets = plain_order(s["idx"], case["E"])
    token = torch.div(route_of, case["K"], rounding_mode="floor").clamp(min=0).long()
    here = (route_of >= 0)[:, None]
    got = {"row_of": row_of, "route_of": route_of, "offsets": offsets}
    if case["dtype"] == "fp8":
        rows = torch.where(here, x.view(torch.uint8)[token], torch.zeros((), dtype=torch.uint8, device=x.device))
        got["rows"] = rows.view(torch.float8_e4m3fn)
        got["scale"] = torch.where(here, s["scale"][token], torch.zeros((), device=x.device))
        return got
    got["rows"] = torch.where(here, x[token], torch.zeros((), dtype=x.dtype, device=x.device))
    if case["grad"]:
        back = s["grad"].float()[row_of.clamp(min=0).long()]
        got["x_grad"] = torch.where((row_of >= 0)[..., None], back, torch.zeros((), device=x.device)).sum(1).to(x.dtype)
    return got


def plain_unsort(s):
    case, rows, weight = s["case"], s["rows"].detach(), s["weight"].detach()
    zero = torch.zeros((), device=rows.device)
    here = s["row_of"] >= 0
    taken = torch.where(here[..., None], rows.float()[s["row_of"].clamp(min=0).long()], zero)
    out = (taken * weight[..., None]).sum(1)
    if case["residual"]:
        out = out + s["residual"].float()
    got = {"out": out.to(DTYPES[case["out"]])}
    if case["grad"]:
        g = s["grad"].float()
        got["weight_grad"] = (taken * g[:, None, :]).sum(2)
        route = s["route_of"].clamp(min=0).long()
        back = weight.reshape(-1)[route][:, None] * g[torch.div(route, case["K"], rounding_mode="floor")]
        got["rows_grad"] = torch.where((s["route_of"] >= 0)[:, None], back, zero).to(rows.dtype)
    return got


def plain_int4(s):
    case = s["case"]
    E, N, K, C = case["E"], case["N"], case["K"], s["most"]
    q = torch.stack((s["q"] & 15, s["q"] >> 4), dim=3).view(E, N, K // case["group"], case["group"]).float()
    q -= 8.0 if s["zero"] is None else s["zero"].float()[..., None]
    q *= s["wscale"].float()[..., None]
    x = s["x"].float()
    if s["scale"] is not None:
        x = x * s["scale"].repeat_interleave(QBLOCK, dim=1)[:, :K]
    R = x.shape[0]
    # every expert's rows, padded to the longest, times its weights
    first = s["offsets"][:-1].long()[:, None]
    at = first + torch.arange(C, device=x.device)
    there = at < s["offsets"][1:].long()[:, None]
    y = torch.bmm(torch.where(there[..., None], x[at.clamp(max=R - 1)], torch.zeros((), device=x.device)),
                  q.view(E, N, K).transpose(1, 2))
    if case["swiglu"]:
        up, gate = y[..., :N // 2], y[..., N // 2:]
        y = gate / (1.0 + torch.exp(-gate)) * up
    out = torch.zeros(R + 1, y.shape[2], device=x.device)
    out[torch.where(there, at, torch.full_like(at, R)).view(-1)] = y.reshape(E * C, -1)
    return {"out": out[:R].to(torch.bfloat16 if case["dtype"] == "fp8" else s["x"].dtype)}


# ---- the framework's operators --------------------------------------------------------------------------


def own_norm(s):
    from constellation_b200.context import add_rms_norm, add_rms_norm_fp8

    if s["case"]["out8"]:
        q, scale, kept = add_rms_norm_fp8(s["x"], s["residual"], s["weight"], EPS)
        return {"out": q, "scale": scale, "sum": kept}
    out, kept = add_rms_norm(s["x"], s["residual"], s["weight"], EPS)
    return {"out": out, "sum": kept}


def own_sort(s):
    from constellation_b200.token_sort import sort_routes, sort_tokens

    case = s["case"]
    order = sort_routes(s["idx"], case["E"])
    got = {"row_of": order.row_of, "route_of": order.route_of, "offsets": order.offsets}
    if case["dtype"] == "fp8":
        got["rows"], got["scale"] = sort_tokens(s["x"], order, scale=s["scale"])
        return got
    rows = sort_tokens(s["x"], order)
    if case["grad"]:
        got["x_grad"], = torch.autograd.grad(rows, (s["x"],), s["grad"])
    got["rows"] = rows
    return got


def own_unsort(s):
    from constellation_b200.token_sort import TokenOrder, unsort_tokens

    case = s["case"]
    order = TokenOrder(s["row_of"], s["route_of"], s["offsets"])
    out = unsort_tokens(s["rows"], order, s["weight"], residual=s["residual"], out_dtype=DTYPES[case["out"]])
    got = {"out": out}
    if case["grad"]:
        got["rows_grad"], got["weight_grad"] = torch.autograd.grad(out, (s["rows"], s["weight"]), s["grad"])
    return got


def own_int4(s):
    from constellation_b200.int4 import grouped_int4

    return {"out": grouped_int4(s["x"], s["w"], s["offsets"], x_scale=s["scale"])}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": own_norm, "sort": own_sort, "unsort": own_unsort, "int4": own_int4}[op](state)
    return {"norm": plain_norm, "sort": plain_sort, "unsort": plain_unsort, "int4": plain_int4}[op](state)


# ---- the definitions in 64 bits -------------------------------------------------------------------------


def exact_norm(case, s):
    h = s["x"].double()
    if case["residual"]:
        h += s["residual"].double()
    y = h / (h.square().mean(1, keepdim=True) + EPS).sqrt() * s["weight"].double()
    kept = h if case["residual"] else None
    if not case["out8"]:
        return {"out": y, "sum": kept}
    T, H = y.shape
    scale = torch.stack([part.abs().amax(1) / FP8_MAX for part in y.split(QBLOCK, dim=1)], dim=1)
    scale[scale == 0] = 1.0
    # before its rounding to e4m3
    return {"out": y / scale[:, torch.arange(H, device=y.device) // QBLOCK], "scale": scale, "sum": kept}


def exact_order(idx, E):
    """Routes of one expert after the other, counted on the host."""
    flat = idx.cpu().reshape(-1).tolist()
    of = [[] for _ in range(E)]
    for i, e in enumerate(flat):
        if 0 <= e < E:
            of[e].append(i)
    route = [i for e in of for i in e]
    offsets = [0]
    for e in of:
        offsets.append(offsets[-1] + len(e))
    return torch.tensor(route, dtype=torch.long, device=idx.device), offsets


def exact_sort(case, s):
    route, _ = exact_order(s["idx"], case["E"])
    K, x = case["K"], s["x"].detach().double()
    total = case["T"] * K
    rows = torch.zeros(total, case["H"], dtype=torch.float64, device=x.device)
    rows[:route.numel()] = x[route // K]
    got = {"rows": rows, "row_of": None, "route_of": None, "offsets": None}
    if case["dtype"] == "fp8":
        got["scale"] = torch.zeros(total, s["scale"].shape[1], dtype=torch.float64, device=x.device)
        got["scale"][:route.numel()] = s["scale"].double()[route // K]
    if case["grad"]:
        got["x_grad"] = torch.zeros_like(x).index_add_(0, route // K, s["grad"][:route.numel()].double())
    return got


def exact_unsort(case, s):
    rows, weight, K = s["rows"].detach().double(), s["weight"].detach().double(), case["K"]
    out = s["residual"].double() if case["residual"] else torch.zeros(case["T"], case["H"], dtype=torch.float64,
                                                                       device=rows.device)
    got = {"out": out}
    g = s["grad"].double() if case["grad"] else None
    if case["grad"]:
        got["weight_grad"], got["rows_grad"] = torch.zeros_like(weight), torch.zeros_like(rows)
    for k in range(K):
        t = (s["row_of"][:, k] >= 0).nonzero().view(-1)
        r = s["row_of"][t, k].long()
        out[t] += weight[t, k, None] * rows[r]
        if case["grad"]:
            got["weight_grad"][t, k] = (rows[r] * g[t]).sum(1)
            got["rows_grad"][r] = weight[t, k, None] * g[t]
    return got


def exact_int4(case, s):
    N, K, group = case["N"], case["K"], case["group"]
    R = s["x"].shape[0]
    out = torch.zeros(R, N // 2 if case["swiglu"] else N, dtype=torch.float64, device="cuda")
    at = s["offsets"].tolist()
    for e in range(case["E"]):
        if at[e] == at[e + 1]:
            continue
        w = torch.empty(N, K, dtype=torch.float64, device="cuda")
        w[:, 0::2] = (s["q"][e] % 16).double()
        w[:, 1::2] = (s["q"][e] // 16).double()
        zero = 8.0 if s["zero"] is None else s["zero"][e].double().repeat_interleave(group, 1)
        w = (w - zero) * s["wscale"][e].double().repeat_interleave(group, 1)
        x = s["x"][at[e]:at[e + 1]].double()
        if s["scale"] is not None:
            x = x * s["scale"][at[e]:at[e + 1]].double()[:, torch.arange(K, device="cuda") // QBLOCK]
        y = x @ w.T
        if case["swiglu"]:
            y = y[:, :N // 2] * y[:, N // 2:] * torch.sigmoid(y[:, N // 2:])
        out[at[e]:at[e + 1]] = y
    return {"out": out}


def exact(case, seed):
    global own
    was, own = own, False  # the inputs as the checkpoint has them, not the framework's layout
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"norm": exact_norm, "sort": exact_sort, "unsort": exact_unsort, "int4": exact_int4}[case["op"]](case, s)

"""The mixture-of-experts operators of eval_test_b200.moe, measured: the router with its plan of sorted copies, tokens sorted
by expert and back with their gradients, and the experts' NVFP4 products of tokens routed on the device.

T tokens choose k of E experts; a copy is one (token, choice) pair, and the copies are sorted stably by expert.
"""
import math

import torch

own = False

F32, F16, BF16 = "float32", "float16", "bfloat16"


def listed():
    return [
        # the router of one decoded token
        {"name": "route_token", "op": "route", "T": 1, "E": 128, "k": 8, "type": BF16, "renorm": True, "grad": False, "drop": 0.0},
        # a serving batch
        {"name": "route_serve", "op": "route", "T": 256, "E": 256, "k": 8, "type": F32, "renorm": True, "grad": False, "drop": 0.0},
        # a training batch with padded sequences, and the router's gradient
        {"name": "route_train", "op": "route", "T": 16384, "E": 128, "k": 4, "type": BF16, "renorm": False, "grad": True, "drop": 0.1},
        # tokens to experts and back in a decode step
        {"name": "permute_decode", "op": "permute", "T": 8, "H": 7168, "E": 64, "k": 8, "type": BF16, "grad": False, "drop": 0.0},
        # odd sizes, choices that were dropped
        {"name": "permute_ragged", "op": "permute", "T": 1777, "H": 1001, "E": 17, "k": 3, "type": F16, "grad": True, "drop": 0.1},
        # 32-bit activations, few large experts
        {"name": "permute_f32", "op": "permute", "T": 4096, "H": 2048, "E": 8, "k": 2, "type": F32, "grad": True, "drop": 0.0},
        # a training batch, forwards and backwards
        {"name": "permute_train", "op": "permute", "T": 16384, "H": 4096, "E": 64, "k": 8, "type": BF16, "grad": True, "drop": 0.0},
        # one decoded token: k experts' weights are streamed for it
        {"name": "experts_token", "op": "experts", "T": 1, "E": 64, "k": 8, "N": 4096, "K": 7168, "type": BF16, "gated": False, "drop": 0.0},
        # a decode batch through the gated projections
        {"name": "experts_decode", "op": "experts", "T": 64, "E": 64, "k": 4, "N": 2048, "K": 4096, "type": BF16, "gated": True, "drop": 0.0},
        # small ragged experts, choices that were dropped
        {"name": "experts_ragged", "op": "experts", "T": 333, "E": 16, "k": 2, "N": 640, "K": 768, "type": F32, "gated": False, "drop": 0.1},
        # about 128 rows for each of 64 experts
        {"name": "experts_chunk", "op": "experts", "T": 1024, "E": 64, "k": 8, "N": 4096, "K": 7168, "type": BF16, "gated": False, "drop": 0.0},
        # a prefill batch through the gated projections
        {"name": "experts_prefill", "op": "experts", "T": 4096, "E": 64, "k": 8, "N": 2048, "K": 7168, "type": F16, "gated": True, "drop": 0.0},
    ]


def draw(rng):
    def logarithmic(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("route", "permute", "experts"))
    case = {"op": op, "type": rng.choice((F32, F16, BF16)), "drop": rng.choice((0.0, 0.0, 0.1, 0.5))}
    if op == "route":
        T, E = logarithmic(1, 16384), logarithmic(8, 512)
        T = max(1, min(T, 16384 * 128 // E))
        case |= {"T": T, "E": E, "k": rng.randint(1, min(E, 16)), "renorm": rng.random() < 0.5, "grad": rng.random() < 0.5}
    elif op == "permute":
        k, H = rng.randint(1, 8), logarithmic(64, 8192)
        if rng.random() < 0.6:
            H = H // 64 * 64
        T = max(1, min(logarithmic(1, 16384), 16384 * 4096 * 8 // (k * H * (2 if case["type"] == F32 else 1))))
        case |= {"T": T, "H": H, "E": logarithmic(k, 256), "k": k, "grad": rng.random() < 0.6}
    else:
        k, E = rng.randint(1, 8), logarithmic(8, 64)
        N, K = 128 * rng.randint(1, 32), 256 * rng.randint(1, 28)
        gated = rng.random() < 0.5
        T = max(1, min(logarithmic(1, 4096), 4096 * 8 // k))
        while E * N * K * (2 if gated else 1) > 64 * 4096 * 7168 or T * k * N * K * (2 if gated else 1) > 32768 * 4096 * 7168:
            N = max(128, N // 256 * 128)
        case |= {"T": T, "E": E, "k": k, "N": N, "K": K, "gated": gated}
    return case


# ------------------------------------------------------------------------------------------------ inputs
def _choices(T, E, k, drop, gen):
    """Choices of a router whose experts are not equally liked: [T, k], none twice in a token; a dropped one is -1."""
    like = torch.randn((1, E), generator=gen, device="cuda") * 0.4
    score = torch.randn((T, E), generator=gen, device="cuda") + like
    ids = score.topk(k, dim=1).indices.int()
    if drop:
        ids = torch.where(torch.rand((T, k), generator=gen, device="cuda") < drop, -1, ids)
    weights = torch.rand((T, k), generator=gen, device="cuda") + 0.05
    return ids.contiguous(), (weights / weights.sum(1, keepdim=True)).contiguous()


def _weights(E, N, K, gen):
    """Expert weights as a checkpoint holds them: packed e2m1 codes [E, N, K/2] of about normal values, and e4m3 scales
    in 128 x 4 tiles, [E, N/128, K/64, 512] bytes."""
    # sixteen equally likely codes whose magnitudes are spread as those of a normal block over its largest value
    spread = torch.tensor([0, 1, 1, 2, 3, 4, 5, 7, 8, 9, 9, 10, 11, 12, 13, 15], dtype=torch.uint8, device="cuda")
    pairs = (spread[:, None] << 4 | spread[None, :]).reshape(256)
    codes = pairs[torch.randint(0, 256, (E, N, K // 2), generator=gen, device="cuda", dtype=torch.int32)]
    scales = (torch.rand((E, N // 128, K // 64, 512), generator=gen, device="cuda") * 0.4 + 0.2).to(torch.float8_e4m3fn)
    return codes, scales.view(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = getattr(torch, case["type"])
    T, E, k = case["T"], case["E"], case["k"]
    s = dict(case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    if case["op"] == "route":
        s["logits"] = (torch.randn((T, E), generator=gen, device="cuda") * 1.5 +
                       torch.randn((1, E), generator=gen, device="cuda") * 0.4).to(dtype)
        s["mask"] = torch.rand((T,), generator=gen, device="cuda") >= case["drop"] if case["drop"] else None
        s["dw"] = torch.randn((T, k), generator=gen, device="cuda")
        return s
    s["experts"], s["weights"] = _choices(T, E, k, case["drop"], gen)
    if case["op"] == "permute":
        H = case["H"]
        s["x"], s["y"] = normal(T, H), normal(T * k, H)
        if case["grad"]:
            s["dout"], s["dxs"] = normal(T, H), normal(T * k, H)
        return s
    N, K = case["N"], case["K"]
    s["x"] = normal(T, K)
    s["w"], s["sw"] = _weights(E, N, K, gen)
    if case["gated"]:
        s["w2"], s["sw2"] = _weights(E, N, K, gen)
    s["alpha"] = torch.rand((E,), generator=gen, device="cuda") * 0.02 + 0.01     # the experts' global scales
    if case["gated"]:
        s["alpha"] = s["alpha"] * 2
    s["most"] = int(torch.bincount(s["experts"][s["experts"] >= 0].long(), minlength=E).max()) if T else 0
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_plan(experts, E):
    flat = experts.reshape(-1).long()
    key = torch.where(flat < 0, E, flat)
    order = torch.sort(key, stable=True).indices
    count = torch.zeros(E + 1, dtype=torch.int64, device=flat.device).scatter_add_(0, key, torch.ones_like(key))[:E]
    offsets = torch.cat([torch.zeros_like(count[:1]), count.cumsum(0)])
    at = torch.empty_like(order)
    at[order] = torch.arange(order.numel(), device=order.device)
    rows = torch.where(flat < 0, -1, at).view(experts.shape)
    source = torch.where(torch.arange(order.numel(), device=order.device) < offsets[-1], order, -1)
    return offsets, rows, source


def _plain_route(s):
    l = s["logits"].float()
    out = torch.isnan(l) | (l == -math.inf)
    if s["mask"] is not None:
        out = out | ~s["mask"][:, None]
    l = torch.where(out, -math.inf, l)
    v, e = torch.sort(l, dim=1, descending=True, stable=True)
    v, e = v[:, :s["k"]], e[:, :s["k"]]
    kept = v > -math.inf
    top = torch.where(kept[:, :1], v[:, :1], 0.0)
    p, pv = torch.exp(l - top), torch.exp(v - top)
    total = pv.sum(1, keepdim=True) if s["renorm"] else p.sum(1, keepdim=True)
    total = torch.where(kept[:, :1], total, 1.0)
    w = torch.where(kept, pv / total, 0.0)
    experts = torch.where(kept, e, -1)
    offsets, rows, source = _plain_plan(experts, s["E"])
    got = {"weights": w, "experts": experts.int(), "offsets": offsets.int(), "rows": rows.int(), "source": source.int()}
    if s["grad"]:
        dw = torch.where(kept, s["dw"], 0.0)
        dot = (w * dw).sum(1, keepdim=True)
        if s["renorm"]:
            d = torch.zeros_like(l).scatter_add_(1, e, w * (dw - dot))
        else:
            d = torch.zeros_like(l).scatter_add_(1, e, dw)
            d = p / total * (d - dot)
        got["dlogits"] = d.to(s["logits"].dtype)
    return got


def _plain_permute(s):
    offsets, rows, source = _plain_plan(s["experts"], s["E"])
    T, k, H = s["T"], s["k"], s["H"]
    kept, at = (rows >= 0)[..., None], rows.clamp(min=0)
    live = (source >= 0)[:, None]
    xs = torch.where(live, s["x"][source.clamp(min=0) // k], 0)
    w = torch.where(rows >= 0, s["weights"], 0.0)
    y = torch.where(kept, s["y"][at], 0).float()
    got = {"xs": xs, "out": (w[..., None] * y).sum(1).to(s["x"].dtype)}
    if s["grad"]:
        dout = s["dout"].float()
        got["dw"] = (dout[:, None, :] * y).sum(2)
        scaled = w.reshape(-1)[source.clamp(min=0)][:, None] * dout[source.clamp(min=0) // k]
        got["dy"] = torch.where(live, scaled, 0.0).to(s["x"].dtype)
        got["dx"] = torch.where(kept, s["dxs"][at], 0).float().sum(1).to(s["x"].dtype)
    return got


def _e2m1(codes):
    """[..., K/2] bytes -> fp32 [..., K], element 2i in the low nibble of byte i."""
    c = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    m = (c & 7).float()
    v = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2, 2 * m - 8))
    return torch.where(c > 7, -v, v)


def _plain_weights(codes, tiled):
    """fp32 [E, N, K] of packed codes and scales in 128 x 4 tiles: row r, block b of a tile is byte
    (r % 32) * 16 + (r / 32) * 4 + b."""
    E, N, _ = codes.shape
    t = tiled.view(E, N // 128, -1, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(E, N, -1)
    s = t.contiguous().view(torch.float8_e4m3fn).float()
    v = _e2m1(codes)
    return v.view(E, N, -1, 16).mul_(s[..., None]).view(E, N, -1)


def _plain_quantised(x):
    """The values that fp32 [T, K] stands for after quantisation to NVFP4: per block of 16 the scale is
    e4m3(min(amax * fl(1/6), 448)), the values are e2m1(x * fl(1/scale)), both to nearest even."""
    b = x.float().view(x.shape[0], -1, 16)
    scale = (b.abs().amax(-1) * torch.tensor(1.0 / 6.0, dtype=torch.float32, device=x.device)).clamp(max=448.0)
    scale = scale.to(torch.float8_e4m3fn).float()[..., None]
    q = torch.where(scale > 0, b * torch.reciprocal(scale), 0.0)
    m = q.abs()
    v = ((m > 0.25).float() + (m >= 0.75).float() + (m > 1.25).float() + (m >= 1.75).float()) * 0.5
    v = v + (m > 2.5).float() + (m >= 3.5).float() + 2 * (m > 5).float()
    return (torch.where(q < 0, -v, v) * scale).view(x.shape)


def _plain_experts(s):
    E, k, alpha = s["E"], s["k"], s["alpha"][:, None, None]
    offsets, _, source = _plain_plan(s["experts"], E)
    C = source.numel()
    r = torch.arange(C, device=source.device)
    live = (r < offsets[-1])[:, None]
    e = torch.searchsorted(offsets[1:], r, right=True).clamp(max=E - 1)
    rows = torch.where(live, _plain_quantised(s["x"])[source.clamp(min=0) // k], 0.0)
    few = C <= E                                     # fewer copies than experts: only the chosen experts' weights
    if few:
        a, slot, take = rows[:, None, :], r, e
    else:                                            # every expert's rows padded to those of the fullest one
        slot = torch.where(live[:, 0], e * s["most"] + (r - offsets[e]), E * s["most"])
        a = torch.zeros((E * s["most"] + 1, s["K"]), device=rows.device)
        a[slot] = rows
        a, take = a[:-1].view(E, s["most"], s["K"]), slice(None)
        slot = slot.clamp(max=max(E * s["most"] - 1, 0))
    c = torch.bmm(a, _plain_weights(s["w"][take], s["sw"][take]).transpose(1, 2)) * alpha[take]
    if s["gated"]:
        c = c / (1 + torch.exp(-c)) * (torch.bmm(a, _plain_weights(s["w2"][take], s["sw2"][take]).transpose(1, 2)) * alpha[take])
    c = c.reshape(-1, s["N"])
    return {"y": (torch.where(live, c[slot], 0.0) if s["most"] else rows.new_zeros((C, s["N"]))).half()}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_route(s):
    from eval_test_b200 import moe
    r = moe.route(s["logits"], s["k"], renormalize=s["renorm"], mask=s["mask"])
    got = {"weights": r.weights, "experts": r.experts, "offsets": r.plan.offsets, "rows": r.plan.rows, "source": r.plan.source}
    if s["grad"]:
        got["dlogits"] = moe.route_backward(s["dw"], s["logits"], r.weights, r.experts, renormalize=s["renorm"])
    return got


def _own_permute(s):
    from eval_test_b200 import moe
    plan = moe.plan(s["experts"], s["E"])
    got = {"xs": moe.dispatch(s["x"], plan), "out": moe.combine(s["y"], plan, s["weights"])}
    if s["grad"]:
        got["dy"], got["dw"] = moe.combine_backward(s["dout"], s["y"], plan, s["weights"])
        got["dx"] = moe.dispatch_backward(s["dxs"], plan)
    return got


def _own_operand(codes, tiled):
    """The framework's view of an operand [rows, K/2, E] and of its scales [32, 4, rows/128, 4, K/64, E]."""
    E, N, half = codes.shape
    return (codes.permute(1, 2, 0).view(torch.float4_e2m1fn_x2),
            tiled.view(torch.float8_e4m3fn).view(E, N // 128, half // 32, 32, 4, 4).permute(3, 4, 1, 5, 2, 0))


def _own_experts(s):
    from eval_test_b200 import moe
    plan = moe.plan(s["experts"], s["E"])
    a, sfa = moe.dispatch_nvfp4(s["x"], plan)
    b, sfb = _own_operand(s["w"], s["sw"])
    if not s["gated"]:
        return {"y": moe.expert_gemm(a, sfa, b, sfb, plan, alpha=s["alpha"])}
    b2, sfb2 = _own_operand(s["w2"], s["sw2"])
    return {"y": moe.expert_dual_gemm(a, sfa, b, sfb, b2, sfb2, plan, alpha=s["alpha"])}


def run(state):
    if own:
        return {"route": _own_route, "permute": _own_permute, "experts": _own_experts}[state["op"]](state)
    return {"route": _plain_route, "permute": _plain_permute, "experts": _plain_experts}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ what a pass has to do
def work(case):
    size = 4 if case["type"] == F32 else 2
    T, E, k = case["T"], case["E"], case["k"]
    C = T * k
    plan = C * 8 + (E + 1) * 4                       # rows and sources, first rows
    if case["op"] == "route":
        grad = case["grad"]
        return {"bytes": T * E * size * (2 if grad else 1) + C * (12 if grad else 8) + plan + (T if case["drop"] else 0),
                "flops": T * E * (8 if grad else 4)}
    live = C * (1 - case["drop"])
    if case["op"] == "permute":
        H = case["H"]
        grad = case["grad"]
        # x -> xs, y -> out; the gradient: dout -> dy (y is read once), dxs -> dx
        return {"bytes": C * 8 + plan + (T + C + live + T) * H * size + ((T + C + live + T) * H * size + C * 4 if grad else 0),
                "flops": live * H * (2 + (4 if grad else 0))}
    N, K, pair = case["N"], case["K"], 2 if case["gated"] else 1
    active = E * (1 - (1 - k * (1 - case["drop"]) / E) ** T)
    return {"bytes": C * 4 + plan + T * K * size + active * N * K * 9 / 16 * pair + C * N * 2,
            "flops": 2 * live * N * K * pair}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    T, E, k = s["T"], s["E"], s["k"]
    dev = "cuda"
    if s["op"] == "route":
        l = s["logits"].double()
        if s["mask"] is not None:
            l[~s["mask"]] = -math.inf
        l[torch.isnan(l)] = -math.inf
        w = torch.zeros((T, k), dtype=torch.float64, device=dev)
        e = torch.full((T, k), -1, dtype=torch.int64, device=dev)
        left = l.clone()
        index = torch.arange(E, device=dev)
        for j in range(k):                            # the largest that is left, the lowest index of equal ones
            best = left.amax(1, keepdim=True)
            at = torch.where(left == best, index, E).amin(1)
            e[:, j] = torch.where(best[:, 0] > -math.inf, at, -1)
            left.scatter_(1, at[:, None], -math.inf)
        chosen = torch.zeros((T, E + 1), dtype=torch.bool, device=dev).scatter_(1, torch.where(e < 0, E, e), True)[:, :E]
        p = torch.where(chosen, l, -math.inf) if s["renorm"] else l
        any_ = (e[:, :1] >= 0)
        p = torch.where(any_, torch.softmax(torch.where(any_, p, 0.0), dim=1), 0.0)
        w = torch.where(e < 0, 0.0, p.gather(1, e.clamp(min=0)))
        got = {"weights": w, "experts": None, "offsets": None, "rows": None, "source": None}
        if s["grad"]:
            g = torch.zeros((T, E + 1), dtype=torch.float64, device=dev)
            g.scatter_(1, torch.where(e < 0, E, e), s["dw"].double())
            g = g[:, :E]
            got["dlogits"] = p * (g - (p * g).sum(1, keepdim=True))
        return got
    ids = s["experts"].reshape(-1)
    source = torch.cat([(ids == e).nonzero()[:, 0] for e in range(E)])
    C, live = T * k, source.numel()
    if s["op"] == "permute":
        H = s["H"]
        w = s["weights"].double().reshape(-1)
        xs = torch.zeros((C, H), dtype=torch.float64, device=dev)
        xs[:live] = s["x"][source // k].double()
        out = torch.zeros((T, H), dtype=torch.float64, device=dev)
        out.index_add_(0, source // k, s["y"][:live].double() * w[source][:, None])
        got = {"xs": xs, "out": out}
        if s["grad"]:
            # (sums of one token's copies are taken in any order: 64 bits hold them)
            dw = torch.zeros(C, dtype=torch.float64, device=dev)
            d = s["dout"].double()[source // k]
            dw[source] = torch.linalg.vecdot(d, s["y"][:live].double())
            d *= w[source][:, None]
            got["dw"] = dw.view(T, k)
            got["dy"] = torch.zeros((C, H), dtype=torch.float64, device=dev)
            got["dy"][:live] = d
            got["dx"] = torch.zeros((T, H), dtype=torch.float64, device=dev)
            got["dx"].index_add_(0, source // k, s["dxs"][:live].double())
        return got
    # the quantiser's two products and its reciprocal are fp32 roundings by definition; what follows has none
    K, N = s["K"], s["N"]
    values = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=dev)
    b = s["x"].double().view(T, K // 16, 16)
    sixth = torch.tensor(1 / 6, dtype=torch.float32, device=dev).double()
    scale = (b.abs().amax(2) * sixth).float().clamp(max=448.0).to(torch.float8_e4m3fn).double()
    inverse = torch.where(scale > 0, 1 / scale, 0.0).float().double()
    q = (b * inverse[..., None]).float().double()
    border = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5], dtype=torch.float64, device=dev)
    low = torch.searchsorted(border, q.abs().contiguous())                 # a value on a border stays below it ...
    tie = (q.abs() == border[low.clamp(max=6)]) & (low < 7) & (low % 2 == 1)   # ... unless the code above it is the even one
    a = (values[low + tie] * torch.sign(q) * scale[..., None]).view(T, K)
    y = torch.zeros((C, N), dtype=torch.float64, device=dev)
    r, blk = torch.arange(N, device=dev)[:, None], torch.arange(K // 16, device=dev)[None, :]
    byte = (r // 128 * (K // 64) + blk // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + blk % 4
    first = 0
    for e in range(E):
        n = int((ids == e).sum())
        if not n:
            continue
        part, both = a[source[first:first + n] // k], []
        for name in ("w", "w2") if s["gated"] else ("w",):
            code = s[name][e].int()
            v = values[torch.stack([code % 16, code // 16], dim=2).view(N, K)]
            sc = s["s" + name][e].reshape(-1)[byte].view(torch.float8_e4m3fn).double()
            both.append(part @ (v.view(N, K // 16, 16) * sc[..., None]).view(N, K).T * s["alpha"][e].double())
        y[first:first + n] = both[0] * torch.sigmoid(both[0]) * both[1] if s["gated"] else both[0]
        first += n
    return {"y": y}

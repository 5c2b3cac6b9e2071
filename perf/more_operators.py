"""A mixture-of-experts layer around 8-bit integer products on one MI355X: routing, tokens to their experts and back, gradients,
products of quantized rows.

``listed()`` holds the fixed cases, ``draw(rng)`` more of the same kinds over the whole range of sizes. A case is a dict of
plain values; ``prepare`` makes its inputs on the GPU from a seed, ``run`` makes one pass: with ``own`` false in plain torch,
with ``own`` true through the public entry points of ``brimkern_amd.Context``; ``exact`` computes the same outputs in 64 bits.
Kinds (T tokens, E experts, k of them for each token, rows of H values):

``route``    logits [T, E] to the k best experts of every token and their weights, and the assignments sorted by expert
``spread``   the tokens' rows copied to their experts' rows, and the experts' outputs back to the tokens, weighted and summed
``grad``     the gradient of both: of the experts' rows, of the weights, of the logits and of the tokens
``i8``       rows quantized to 8 bits, a scale each, times an 8-bit weight [N, K] with a scale for every channel
``i8moe``    the same by experts: weights [E, N, K], the rows of the tokens found by index (``gather``), or rows that lie sorted
             and are made of a gate and an up projection on the way (``glu``)

An assignment is a pair (token, place among its k); sorted rows are the assignments ordered by expert, then by token and place.
Assignments to experts outside [0, E) (held by another device) have no row.

The library's context has a stream of its own, which does not wait for torch's and which torch's does not wait for. So with
``own`` true ``prepare`` returns when its inputs are there; what ``run`` returns is there after ``context().sync()`` (or
``torch.cuda.synchronize()``, which waits for every stream), and a state is kept until then.
"""
import math

import torch

DEV = "cuda:0"
own = False

_context = None


def context():
    """The one library context of the process (a program keeps it for its lifetime)."""
    global _context
    if _context is None:
        from brimkern_amd import Context
        _context = Context(0)
    return _context


def listed():
    return [
        # a decoding step of 64 sequences: 8 of 64 experts each
        {"name": "route_decode_64", "kind": "route", "T": 64, "E": 64, "k": 8, **_scores()},
        # prompts: many experts, sigmoid scores with a bias that evens the load out
        {"name": "route_prompt_16384", "kind": "route", "T": 16384, "E": 256, "k": 8, **_scores(sigmoid=True, bias=True, scale=2.5)},
        # a step of 256 tokens
        {"name": "spread_256x8", "kind": "spread", "T": 256, "E": 64, "k": 8, "H": 2048, "away": 0.0, "res": True},
        # long prompts on a device that holds a quarter of the experts
        {"name": "spread_16384x6_away", "kind": "spread", "T": 16384, "E": 64, "k": 6, "H": 2048, "away": 0.75, "res": True},
        # a short odd batch, softmax over all experts
        {"name": "grad_333x4", "kind": "grad", "T": 333, "E": 40, "k": 4, "H": 1000, "away": 0.0, **_scores(renorm=False)},
        # a training batch
        {"name": "grad_4096x8", "kind": "grad", "T": 4096, "E": 64, "k": 8, "H": 2048, "away": 0.0, **_scores()},
        # one token: the call that a single user waits for
        {"name": "i8_decode_1", "kind": "i8", "M": 1, "K": 2560, "N": 9728, "res": False},
        # a few sequences decoded together, an odd number of channels
        {"name": "i8_decode_24", "kind": "i8", "M": 24, "K": 4096, "N": 2561, "res": True},
        # a prompt of 512 tokens
        {"name": "i8_prompt_512", "kind": "i8", "M": 512, "K": 2560, "N": 9728, "res": False},
        # long prompts: the largest
        {"name": "i8_prompt_8192", "kind": "i8", "M": 8192, "K": 9728, "N": 2560, "res": True},
        # gate and up projections of 256 tokens, 8 of 64 experts each
        {"name": "i8moe_256_gate_up", "kind": "i8moe", "T": 256, "E": 64, "k": 8, "K": 2048, "N": 1536, "gather": True, "glu": False},
        # down projections of a prompt
        {"name": "i8moe_4096_down", "kind": "i8moe", "T": 4096, "E": 64, "k": 8, "K": 768, "N": 2048, "gather": False, "glu": True},
    ]


def _scores(sigmoid=False, renorm=True, bias=False, scale=1.0):
    return {"sigmoid": sigmoid, "renorm": renorm, "bias": bias, "scale": scale}


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


LARGEST = 8192 * 9728 * 2560                  # products of the largest listed case


def draw(rng):
    kind = rng.choice(["route", "spread", "grad", "i8", "i8", "i8", "i8moe", "i8moe"])
    if kind == "i8":
        K = 32 * _log(rng, 2, 320)
        N = _log(rng, 16, 10240)
        M = _log(rng, 1, min(8192, LARGEST // (K * N)))
        return {"kind": kind, "M": M, "K": K, "N": N, "res": rng.random() < 0.3}
    E = rng.choice([4, 8, 16, 40, 64, 64, 100, 128, 256])
    k = rng.choice([1, 2, 4, 6, 8])
    k = min(k, E)
    c = {"kind": kind, "T": _log(rng, 1, 16384), "E": E, "k": k}
    if kind in ("route", "grad"):
        c.update(_scores(rng.random() < 0.4, rng.random() < 0.6, kind == "route" and rng.random() < 0.4, rng.choice([1.0, 1.0, 2.5])))
    if kind == "route":
        return c
    if kind == "i8moe":
        c["K"], c["N"] = 32 * _log(rng, 2, 96), _log(rng, 16, 4096)
        c["E"] = E = max(k, min(E, (1 << 29) // (c["K"] * c["N"])))
        c["T"] = _log(rng, 1, max(1, min(8192, LARGEST // (2 * c["K"] * c["N"] * k))))
        c["gather"] = rng.random() < 0.5
        c["glu"] = not c["gather"]
        return c
    c["H"] = 4 * _log(rng, 16, 1024)
    c["T"] = max(1, min(c["T"], (1 << 26) // (c["H"] * c["k"])))
    c["away"] = rng.choice([0.0, 0.0, 0.5])
    if kind == "spread":
        c["res"] = rng.random() < 0.5
    return c


# ---- inputs --------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _logits(g, c):
    """A router's logits: some experts are liked more by all tokens."""
    return 1.5 * torch.randn(c["T"], c["E"], generator=g, device=DEV) + 0.7 * torch.randn(c["E"], generator=g, device=DEV)


def _ints(v):
    return v.to(torch.int32).contiguous()


def _sorted(ids, E):
    """(row_off, src, slot) of assignments to experts: assignments by row, -1 behind the last; rows by assignment, or -1."""
    flat = ids.flatten().long()
    key = torch.where((flat >= 0) & (flat < E), flat, E)
    src = torch.argsort(key, stable=True)
    row = torch.argsort(src)
    row_off = torch.searchsorted(key[src], torch.arange(E + 1, device=DEV))
    kept = key < E
    src = torch.where(kept[src], src, -1)
    return _ints(row_off), _ints(src), _ints(torch.where(kept, row, -1).view(ids.shape))


def _rows(g, M, K):
    """Activations: normal, with a log-normal gain per channel and a few channels far above the others."""
    gain = torch.exp(0.4 * torch.randn(K, generator=g, device=DEV))
    gain[torch.randperm(K, generator=g, device=DEV)[: max(1, K // 500)]] *= 12
    return torch.randn(M, K, generator=g, device=DEV) * gain


def _weight(g, *shape):
    """8-bit codes [.., N, K] and a scale per channel of them."""
    codes = (torch.randn(*shape, generator=g, device=DEV) * 32).round_().clamp_(-127, 127).to(torch.int8)
    scales = (0.02 + 0.01 * torch.rand(*shape[:-1], generator=g, device=DEV)) / math.sqrt(shape[-1])
    return codes, scales


def _inputs(c, seed):
    """The tensors of a case, from the seed alone."""
    g, kind = _gen(seed), c["kind"]
    if kind == "i8":
        s = {"x": _rows(g, c["M"], c["K"])}
        s["w"], s["ws"] = _weight(g, c["N"], c["K"])
        if c["res"]:
            s["res"] = torch.randn(c["M"], c["N"], generator=g, device=DEV)
        return s
    s = {"logits": _logits(g, c)}
    if c.get("bias"):
        s["bias"] = 0.1 * torch.randn(c["E"], generator=g, device=DEV)
    if kind == "route":
        return s
    T, E, k = c["T"], c["E"], c["k"]
    s["ids"] = _ints(torch.sort(s["logits"], dim=-1, descending=True, stable=True)[1][:, :k])
    if c.get("away"):
        # experts from E - away E on are another device's: assignments to them have no row here
        s["ids"] = torch.where(s["ids"] >= E - int(c["away"] * E), -1, s["ids"])
    s["row_off"], s["src"], s["slot"] = _sorted(s["ids"], E)
    if kind == "i8moe":
        s["w"], s["ws"] = _weight(g, E, c["N"], c["K"])
        s["x"] = _rows(g, T, c["K"]) if c["gather"] else torch.randn(T * k, 2 * c["K"], generator=g, device=DEV)
        return s
    H = c["H"]
    if kind == "spread":
        s["weights"] = torch.softmax(torch.randn(T, k, generator=g, device=DEV), -1)
        s["x"], s["y"] = torch.randn(T, H, generator=g, device=DEV), torch.randn(T * k, H, generator=g, device=DEV)
        s["res"] = torch.randn(T, H, generator=g, device=DEV) if c["res"] else None
        return s
    s["weights"] = _plain_weights(c, s["logits"], s["ids"])
    s["dout"] = torch.randn(T, H, generator=g, device=DEV)
    s["y"], s["dx_sorted"] = (torch.randn(T * k, H, generator=g, device=DEV) for _ in range(2))
    return s


def _at(t):
    return t.data_ptr() if t is not None and t.numel() else None


def prepare(case, seed):
    c, s = case, {**_inputs(case, seed), "case": dict(case)}
    kind = c["kind"]
    empty = lambda *shape, dtype=torch.float32: torch.zeros(*shape, dtype=dtype, device=DEV)
    if kind == "i8":
        s["codes"], s["scales"] = empty(c["M"], c["K"], dtype=torch.int8), empty(c["M"])
        s["out"] = empty(c["M"], c["N"])
    elif kind == "i8moe":
        M = c["T"] if c["gather"] else c["T"] * c["k"]
        s["codes"], s["scales"] = empty(M, c["K"], dtype=torch.int8), empty(M)
        s["out"] = empty(c["T"] * c["k"], c["N"])
        s["most"] = int((s["row_off"][1:] - s["row_off"][:-1]).max())        # rows of an expert: the plain form's batch
    elif kind == "route":
        T, k = c["T"], c["k"]
        s["ids_out"], s["w_out"] = empty(T, k, dtype=torch.int32), empty(T, k)
        s["row_off_out"], s["src_out"] = empty(c["E"] + 1, dtype=torch.int32), empty(T * k, dtype=torch.int32)
        s["slot_out"] = empty(T, k, dtype=torch.int32)
        if own:
            s["args"] = _route_args(s)
    else:
        T, k, H = c["T"], c["k"], c["H"]
        s["rows"], s["out"] = empty(T * k, H), empty(T, H)
        if kind == "grad":
            s["dw"], s["dlogits"] = empty(T, k), empty(T, c["E"])
            if own:
                s["args"] = _route_args(s)
    if own:
        torch.cuda.synchronize()                         # the library's stream does not wait for torch's
    return s


def _route_args(s):
    c, grad = s["case"], s["case"]["kind"] == "grad"
    made = {} if grad else {"row_off": _at(s["row_off_out"]), "src": _at(s["src_out"]), "slot": _at(s["slot_out"])}
    return context().moe_route_args(logits=_at(s["logits"]), tokens=c["T"], experts=c["E"], k=c["k"], bias=_at(s.get("bias")),
                                    ids=_at(s["ids"] if grad else s["ids_out"]), weights=_at(s["weights"] if grad else s["w_out"]),
                                    sigmoid=c["sigmoid"], renorm=c["renorm"], scale=c["scale"], **made)


# ---- one pass ------------------------------------------------------------------------------------


def run(s):
    c, kind = s["case"], s["case"]["kind"]
    if own:
        return _run_own(context(), s, c, kind)
    if kind == "route":
        ids = _choose(c, s["logits"], s.get("bias"))
        row_off, src, slot = _sorted(ids, c["E"])
        return {"ids": ids, "weights": _plain_weights(c, s["logits"], ids), "row_off": row_off, "src": src, "slot": slot}
    if kind == "spread":
        kept = s["slot"] >= 0
        rows = torch.zeros_like(s["rows"])
        rows[s["slot"][kept].long()] = s["x"].repeat_interleave(c["k"], 0)[kept.flatten()]
        back = torch.where(kept[..., None], s["y"][s["slot"].clamp_min(0).long()] * s["weights"][..., None], 0.0).sum(1)
        return {"rows": rows, "out": back if s["res"] is None else s["res"] + back}
    if kind == "grad":
        return _plain_grad(c, s)
    if kind == "i8":
        codes, scales = _quantize(s["x"].double())
        y = (codes.float() @ s["w"].float().t()) * s["ws"] * scales[:, None]
        return y + s["res"] if c["res"] else y
    if c["glu"]:
        gate, up = s["x"].double().chunk(2, -1)
        codes, scales = _quantize(gate / (1 + torch.exp(-gate)) * up)
    else:
        codes, scales = _quantize(s["x"].double())
    return _plain_experts(c, s, codes.float(), scales)


def _run_own(ctx, s, c, kind):
    if kind == "route":
        ctx.moe_route(s["args"])
        return {"ids": s["ids_out"], "weights": s["w_out"], "row_off": s["row_off_out"], "src": s["src_out"], "slot": s["slot_out"]}
    if kind == "spread":
        ctx.moe_dispatch(_at(s["x"]), _at(s["slot"]), None, _at(s["rows"]), c["T"], c["k"], c["H"])
        ctx.moe_combine(_at(s["y"]), _at(s["slot"]), _at(s["weights"]), _at(s["res"]), _at(s["out"]), c["T"], c["k"], c["H"])
        return {"rows": s["rows"], "out": s["out"]}
    if kind == "grad":
        ctx.moe_combine_grad(_at(s["dout"]), _at(s["y"]), _at(s["slot"]), _at(s["weights"]), _at(s["rows"]), _at(s["dw"]), c["T"], c["k"], c["H"])
        ctx.moe_route_grad(s["args"], _at(s["dw"]), _at(s["dlogits"]))
        ctx.moe_combine(_at(s["dx_sorted"]), _at(s["slot"]), None, None, _at(s["out"]), c["T"], c["k"], c["H"])
        return {"dy": s["rows"], "dw": s["dw"], "dlogits": s["dlogits"], "dx": s["out"]}
    K, N = c["K"], c["N"]
    if kind == "i8":
        ctx.quantize_i8(_at(s["x"]), _at(s["codes"]), _at(s["scales"]), c["M"], K)
        ctx.matmul_t_i8(_at(s["codes"]), _at(s["scales"]), _at(s["w"]), _at(s["ws"]), _at(s["out"]), c["M"], K, N, res=_at(s.get("res")))
        return s["out"]
    R = c["T"] * c["k"]
    if c["glu"]:
        # rows of gate and up side by side
        ctx.quantize_i8(_at(s["x"]) + 4 * K, _at(s["codes"]), _at(s["scales"]), R, K, x_stride=2 * K, gate=_at(s["x"]), gate_stride=2 * K)
    else:
        ctx.quantize_i8(_at(s["x"]), _at(s["codes"]), _at(s["scales"]), c["T"], K)
    by = {"src": _at(s["src"]), "k": c["k"]} if c["gather"] else {}
    ctx.moe_matmul_t_i8(_at(s["codes"]), _at(s["scales"]), _at(s["row_off"]), _at(s["w"]), _at(s["ws"]), _at(s["out"]), c["E"], R, K, N, **by)
    return s["out"]


def _choose(c, logits, bias):
    """The k best experts of every token, ties to the lower one."""
    key = logits
    if bias is not None:
        key = (torch.sigmoid(logits.double()) if c["sigmoid"] else torch.softmax(logits.double(), -1)) + bias.double()
    return _ints(torch.sort(key, dim=-1, descending=True, stable=True)[1][:, :c["k"]])


def _plain_weights(c, logits, ids):
    """The weights of chosen experts [T, k]; of none (-1): 0."""
    kept = ids >= 0
    at = ids.clamp_min(0).long()
    if c["sigmoid"]:
        s = 1 / (1 + torch.exp(-logits.double()))
    else:
        e = torch.exp((logits - logits.amax(-1, keepdim=True)).double())
        s = e / e.sum(-1, keepdim=True)
    w = torch.where(kept, s.gather(1, at), 0.0)
    if c["renorm"]:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total == 0, 1.0, total)
    return (w * c["scale"]).float()


def _plain_grad(c, s):
    kept, at = s["slot"] >= 0, s["slot"].clamp_min(0).long()
    rows = torch.zeros_like(s["rows"])
    rows[s["slot"][kept].long()] = (s["dout"][:, None] * s["weights"][..., None])[kept]
    dw = torch.where(kept, (s["dout"][:, None] * s["y"][at]).sum(-1), 0.0)
    # of the logits, by the formulas, in 64 bits
    logits, ids = s["logits"].double(), s["ids"].clamp_min(0).long()
    chosen = s["ids"] >= 0
    g = torch.where(chosen, dw.double(), 0.0) * c["scale"]
    score = 1 / (1 + torch.exp(-logits)) if c["sigmoid"] else torch.softmax(logits, -1)
    sel = torch.where(chosen, score.gather(1, ids), 0.0)
    if c["renorm"]:
        total = sel.sum(-1, keepdim=True)
        total = torch.where(total == 0, 1.0, total)
        g = (g - (sel / total * g).sum(-1, keepdim=True)) / total
    ds = torch.zeros_like(logits).scatter_add_(1, ids, torch.where(chosen, g, 0.0))
    dl = ds * score * (1 - score) if c["sigmoid"] else score * (ds - (ds * score).sum(-1, keepdim=True))
    dx = torch.where(kept[..., None], s["dx_sorted"][at], 0.0).sum(1)
    return {"dy": rows, "dw": dw, "dlogits": dl.float(), "dx": dx}


def _quantize(h):
    """Codes and f32 scales of rows in 64 bits: to the nearest code, ties upward."""
    levels = torch.tensor(127.0, dtype=torch.float64, device=DEV)          # (x / 127.0 would multiply)
    scale = (h.abs().amax(-1) / levels).float()
    step = scale.double()[:, None]
    codes = torch.floor(h / torch.where(step == 0, 1.0, step) + 0.5).clamp_(-127, 127)
    return torch.where(step == 0, 0.0, codes).to(torch.int8), scale


def _plain_experts(c, s, codes, scales):
    """Every expert's rows as a batch of as many rows as the largest has."""
    E, most, off = c["E"], s["most"], s["row_off"].long()
    row = off[:-1, None] + torch.arange(most, device=DEV)
    real = row < off[1:, None]
    row = torch.where(real, row, 0)
    at = s["src"].long()[row] // c["k"] if c["gather"] else row
    y = torch.bmm(codes[at], s["w"].float().transpose(1, 2).contiguous()) * s["ws"][:, None] * scales[at][..., None]
    out = torch.zeros_like(s["out"])
    out[row[real]] = y[real]
    return out


# ---- what a pass cannot do without ---------------------------------------------------------------


def _kept(c):
    """Assignments that have a row, by the case alone."""
    E = c["E"]
    return c["T"] * c["k"] * (E - int(c.get("away", 0.0) * E)) / E


def work(case):
    c, kind = case, case["kind"]
    if kind == "i8":
        M, K, N = c["M"], c["K"], c["N"]
        return {"bytes": 4 * M * K + N * K + 4 * N + 4 * M * N * (2 if c["res"] else 1), "flops": 2 * M * N * K}
    T, E, k = c["T"], c["E"], c["k"]
    if kind == "route":
        return {"bytes": 4 * T * E + 16 * T * k + 4 * E, "flops": 4 * T * E}
    R = _kept(c)
    if kind == "spread":
        return {"bytes": 4 * c["H"] * (2 * T + 2 * R + (T if c["res"] else 0)) + 12 * T * k, "flops": 2 * R * c["H"]}
    if kind == "grad":
        return {"bytes": 4 * c["H"] * (2 * T + 3 * R) + 8 * T * E + 16 * T * k, "flops": 4 * R * c["H"]}
    used = min(E, T * k)                                 # experts that have rows, at most
    rows = 4 * T * c["K"] if c["gather"] else 8 * R * c["K"]
    return {"bytes": rows + used * c["N"] * (c["K"] + 4) + 4 * R * c["N"], "flops": 2 * R * c["K"] * c["N"]}


# ---- the same in 64 bits -------------------------------------------------------------------------


def exact(case, seed):
    c, s, f64 = case, _inputs(case, seed), torch.float64
    kind = c["kind"]
    if kind in ("i8", "i8moe"):
        return _exact_product(c, s)
    T, E, k = c["T"], c["E"], c["k"]
    if kind == "route":
        logits = s["logits"].to(f64)
        score = torch.special.expit(logits) if c["sigmoid"] else torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
        left = score + s["bias"].to(f64) if c["bias"] else logits.clone()
        ids = torch.empty(T, k, dtype=torch.int64, device=DEV)
        for j in range(k):                               # the best, then the best of the others
            best = left.max(-1, keepdim=True)[0]
            ids[:, j] = torch.where(left == best, torch.arange(E, device=DEV), E).min(-1)[0]
            left.scatter_(1, ids[:, j:j + 1], -math.inf)
        w = score.gather(1, ids)
        if c["renorm"]:
            w = w / w.sum(-1, keepdim=True)
        # every assignment's row: those of lower experts, and those before it of its own
        flat = ids.flatten()
        counts = torch.bincount(flat, minlength=E)
        row_off = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
        slot, src = torch.empty_like(flat), torch.empty_like(flat)
        for e in range(E):
            mine = torch.nonzero(flat == e).flatten()
            slot[mine] = row_off[e] + torch.arange(len(mine), device=DEV)
            src[row_off[e]:row_off[e + 1]] = mine
        return {"ids": _ints(ids), "weights": w * c["scale"], "row_off": _ints(row_off), "src": _ints(src), "slot": _ints(slot.view(T, k))}
    H, R = c["H"], T * k
    place = torch.nonzero(s["slot"].flatten() >= 0).flatten()
    row, token = s["slot"].flatten()[place].long(), place // k
    if kind == "spread":
        rows = torch.zeros(R, H, dtype=f64, device=DEV).index_copy_(0, row, s["x"].to(f64)[token])
        out = s["res"].to(f64) if c["res"] else torch.zeros(T, H, dtype=f64, device=DEV)
        out = out.index_add(0, token, s["y"].to(f64)[row] * s["weights"].flatten()[place].to(f64)[:, None])
        return {"rows": rows, "out": out}
    dout = s["dout"].to(f64)
    dy = torch.zeros(R, H, dtype=f64, device=DEV).index_copy_(0, row, dout[token] * s["weights"].flatten()[place].to(f64)[:, None])
    dw = torch.zeros(R, dtype=f64, device=DEV)
    dw[place] = torch.linalg.vecdot(dout[token], s["y"].to(f64)[row])
    dx = torch.zeros(T, H, dtype=f64, device=DEV).index_add_(0, token, s["dx_sorted"].to(f64)[row])
    # of the logits: differentiated by the library, from the weights' own definition
    logits = s["logits"].to(f64).requires_grad_()
    score = torch.sigmoid(logits) if c["sigmoid"] else torch.softmax(logits, -1)
    chosen = s["ids"] >= 0
    w = score.gather(1, s["ids"].clamp_min(0).long()) * chosen
    if c["renorm"]:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(chosen.any(-1, keepdim=True), total, 1.0)
    (dl,) = torch.autograd.grad((w * c["scale"] * dw.view(T, k)).sum(), logits)
    return {"dy": dy, "dw": dw.view(T, k), "dlogits": dl, "dx": dx}


def _exact_product(c, s):
    """The products expert by expert, or piece by piece of the rows, of values (code times scale) in 64 bits."""
    f64, x = torch.float64, s["x"].to(torch.float64)
    if c["kind"] == "i8moe" and c["glu"]:
        x = x[:, :c["K"]] * torch.special.expit(x[:, :c["K"]]) * x[:, c["K"]:]
    scale = (x.abs().max(-1, keepdim=True)[0] / torch.full_like(x[:, :1], 127)).to(torch.float32).to(f64)
    part = x / torch.where(scale == 0, 1.0, scale)
    low = torch.floor(part)
    value = scale * (low + (part - low >= 0.5)).clamp(-127, 127)
    if c["kind"] == "i8":
        w = s["w"].to(f64) * s["ws"].to(f64)[:, None]
        y = torch.cat([piece @ w.t() for piece in value.split(1024)])
        return y + s["res"].to(f64) if c["res"] else y
    out = torch.zeros(c["T"] * c["k"], c["N"], dtype=f64, device=DEV)
    off = s["row_off"].tolist()
    for e in range(c["E"]):
        a, b = off[e], off[e + 1]
        if a < b:
            rows = value[s["src"][a:b].long() // c["k"]] if c["gather"] else value[a:b]
            out[a:b] = rows @ (s["w"][e].to(f64) * s["ws"][e].to(f64)[:, None]).t()
    return out

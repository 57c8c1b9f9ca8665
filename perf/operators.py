"""The expert-layer operators as their users call them: sizes, inputs, plain forms and 64-bit results.

A user who prepares a mixture-of-experts model for error-feedback rounding runs calibration tokens through its expert
layers on the card: the router's logits choose experts and sort the rows by expert (`route`), the stored MXFP4 experts
are multiplied with the rows they received, in the rows' own type or with the rows rounded to MXFP4 too (`matmul`, one
matrix; `experts`, a stack with the rows' grouping, for gate and up together with SwiGLU), and tensors or rows are
rounded to MXFP4, the rounded values coming back for the error sums (`quantize`). Sizes are the benchmark's (experts of
2048 x 7168, 256 and 384 of them, a dense 4096 x 4096), the tests' (1536, 2304 and 1760 columns) and what lies between.

`listed()` are the fixed cases and `draw(rng)` one more of their ranges; `prepare(case, seed)` makes what the user's
program holds before the call, `run(state)` is one pass, in plain torch operations in 32 bits (`own` false) or through
`gpuq.experts` (`own` true), `work(case)` what a pass cannot do without and `exact(case, seed)` its result in 64 bits.
"""
import os
import sys

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2, "mxfp4": 17 / 32}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)         # the magnitudes of e2m1
MIDDLES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)

_lib = []


def lib():
    """the library on the GPU and its module, loaded once a process"""
    if not _lib:
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "trench-gguf_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        import gpuq
        from gpuq import experts
        torch.cuda.init()
        _lib.extend((gpuq.load_gpuq(0), experts))
    return _lib


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one token's activations become MXFP4 ahead of a product: a call whose latency is what counts
        {"name": "quantize_token_bf16", "op": "quantize", "src": "bf16", "rows": 1, "ncol": 7168, "form": "packed"},
        # a float expert is written to a GGUF file as MXFP4 blocks, its rounded values kept for the error report
        {"name": "quantize_expert_f32", "op": "quantize", "src": "f32", "rows": 2048, "ncol": 7168, "form": "blocks"},
        # a stack of 16 BF16 experts, the bulk of a conversion
        {"name": "quantize_experts_bf16", "op": "quantize", "src": "bf16", "rows": 16 * 2048, "ncol": 7168,
         "form": "blocks"},
        # one token through one expert's matrix
        {"name": "matmul_token_bf16", "op": "matmul", "x": "bf16", "m": 1, "ne1": 2048, "ne0": 7168, "out": "f32"},
        # a few rows in full precision through a down projection
        {"name": "matmul_rows_f32", "op": "matmul", "x": "f32", "m": 13, "ne1": 7168, "ne0": 2048, "out": "f32"},
        # a chunk of calibration rows through one matrix, exact weights and BF16 rows
        {"name": "matmul_chunk_bf16", "op": "matmul", "x": "bf16", "m": 4096, "ne1": 2048, "ne0": 7168, "out": "f32"},
        # the same matrix with the rows rounded to MXFP4 on the way, as a server with 4-bit activations would see them
        {"name": "matmul_chunk_mxfp4", "op": "matmul", "x": "mxfp4", "m": 8192, "ne1": 2048, "ne0": 7168,
         "out": "bf16"},
        # a layer's calibration pass: gate and up of 64 experts with SwiGLU, eight experts a token
        {"name": "experts_glu_bf16", "op": "experts", "x": "bf16", "tokens": 4096, "nexp": 64, "topk": 8, "ne1": 2048,
         "ne0": 7168, "glu": True, "out": "bf16"},
        # a few tokens a step against a wide layer: most experts that are read serve a single row
        {"name": "experts_step_bf16", "op": "experts", "x": "bf16", "tokens": 8, "nexp": 256, "topk": 8, "ne1": 2048,
         "ne0": 7168, "glu": False, "out": "f32"},
        # ragged groups of a narrower layer, half-precision rows
        {"name": "experts_ragged_f16", "op": "experts", "x": "f16", "tokens": 999, "nexp": 48, "topk": 6, "ne1": 1536,
         "ne0": 2304, "glu": False, "out": "f32"},
        # the router's choice for one token: sigmoid scores, a balancing bias, 4 of 8 groups
        {"name": "route_token_groups", "op": "route", "logits": "f32", "tokens": 1, "nexp": 256, "topk": 8,
         "score": "sigmoid", "bias": True, "ngroup": 8, "keep": 4, "renorm": True, "scale": 2.5},
        # the choice for a chunk of calibration tokens over 384 experts
        {"name": "route_chunk_softmax", "op": "route", "logits": "bf16", "tokens": 16384, "nexp": 384, "topk": 8,
         "score": "softmax", "bias": False, "ngroup": 1, "keep": 1, "renorm": True, "scale": 1.0},
    ]


def between(rng, lo, hi):
    """a whole number of [lo, hi], spread over its logarithm, odd ones among them"""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["quantize", "quantize", "matmul", "matmul", "matmul", "experts", "experts", "experts", "route",
                     "route"])
    if op == "quantize":
        return {"op": op, "src": rng.choice(["f32", "f16", "bf16"]), "rows": between(rng, 1, 8192),
                "ncol": 32 * between(rng, 1, 225), "form": rng.choice(["blocks", "packed"])}
    if op == "matmul":
        return {"op": op, "x": rng.choice(["bf16", "bf16", "f16", "f32", "mxfp4", "mxfp4"]), "m": between(rng, 1, 4096),
                "ne1": between(rng, 16, 7168), "ne0": 32 * between(rng, 1, 224), "out": rng.choice(["f32", "bf16"])}
    if op == "experts":
        nexp, x = between(rng, 4, 128), rng.choice(["bf16", "bf16", "f16", "f32", "mxfp4"])
        ne1, ne0 = between(rng, 64, 2048), 32 * between(rng, 2, 224)
        while nexp * ne1 * ne0 > 64 * 2048 * 7168:
            nexp = max(4, nexp // 2)
        return {"op": op, "x": x, "tokens": between(rng, 1, 1024 if x == "f32" else 2048),
                "nexp": nexp, "topk": rng.randint(1, min(8, nexp)), "ne1": ne1, "ne0": ne0,
                "glu": rng.random() < 0.5, "out": rng.choice(["f32", "bf16"])}
    ngroup = rng.choice([1, 1, 4, 8])
    nexp = ngroup * between(rng, 4, 384 // ngroup)
    keep = rng.randint(max(1, ngroup // 2), ngroup)
    return {"op": op, "logits": rng.choice(["f32", "f16", "bf16"]), "tokens": between(rng, 1, 16384), "nexp": nexp,
            "topk": rng.randint(1, min(8, keep * (nexp // ngroup))), "score": rng.choice(["softmax", "sigmoid"]),
            "bias": rng.random() < 0.5, "ngroup": ngroup, "keep": keep, "renorm": rng.random() < 0.7,
            "scale": rng.choice([1.0, 2.5])}


def touched(case):
    """the experts that at least one row reaches, on average over evenly used experts"""
    return case["nexp"] * (1 - (1 - case["topk"] / case["nexp"]) ** case["tokens"])


def work(case):
    op = case["op"]
    if op == "quantize":        # the values in, the 17-byte blocks and the rounded BF16 values out
        n = case["rows"] * case["ncol"]
        return {"bytes": int(n * (SIZES[case["src"]] + 17 / 32 + 2)), "flops": 4 * n}
    if op == "route":           # logits in; ids and weights, the experts' offsets and the two row lists out
        n = case["tokens"] * case["topk"]
        return {"bytes": case["tokens"] * case["nexp"] * int(SIZES[case["logits"]]) + 16 * n + 4 * (case["nexp"] + 1),
                "flops": 4 * case["tokens"] * case["nexp"]}
    ne1, ne0 = case["ne1"], case["ne0"]
    mats = 2 if case.get("glu") else 1
    if op == "matmul":
        m, rows, stack = case["m"], case["m"], 1
    else:
        m, rows, stack = case["tokens"], case["tokens"] * case["topk"], touched(case)
    xsize = 2 if case["x"] == "mxfp4" else SIZES[case["x"]]          # (rows rounded on the way arrive as BF16)
    nbytes = m * ne0 * xsize + mats * stack * ne1 * ne0 * 17 / 32 + rows * ne1 * SIZES[case["out"]]
    if op == "experts":
        nbytes += 4 * (rows + case["nexp"] + 1)
    return {"bytes": int(nbytes), "flops": 2 * mats * rows * ne1 * ne0}


# ---------------------------------------------------------------- inputs
def generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE)


def activations(g, rows, ncol, dtype):
    """heavy-tailed rows (Student t of 4 degrees of freedom, as the benchmark's Hessians have), a tenth in size"""
    out = torch.empty((rows, ncol), dtype=dtype, device=DEVICE)
    step = max(1, (1 << 26) // ncol)
    for r in range(0, rows, step):
        n = min(step, rows - r)
        chi = sum(normal(g, n, ncol).square() for _ in range(4))
        out[r:r + n] = (0.1 * normal(g, n, ncol) / (chi / 4).sqrt()).to(dtype)
    return out


def stored_blocks(g, nmat, ne1, ne0):
    """MXFP4 tensors as a GGUF file holds them, [nmat][ne1][ne0 / 32][17] bytes: the benchmark's experts, scale
    exponents uniform in [-8, -4] and uniform codes"""
    b = torch.randint(0, 256, (nmat, ne1, ne0 // 32, 17), generator=g, device=DEVICE, dtype=torch.uint8)
    b[..., 0] = torch.randint(119, 124, b.shape[:-1], generator=g, device=DEVICE, dtype=torch.uint8)
    return b


def grouping(ids, nexp):
    """(offsets [nexp + 1], rows, slots): the assignments sorted by expert, in order within each"""
    flat = ids.reshape(-1)
    by, slots = torch.sort(flat, stable=True)
    offsets = torch.searchsorted(by, torch.arange(nexp + 1, device=flat.device, dtype=flat.dtype))
    return (offsets.to(torch.int32), torch.div(slots, ids.shape[1], rounding_mode="floor").to(torch.int32),
            slots.to(torch.int32))


def router_logits(g, tokens, nexp):
    """logits of a trained router: some experts more used than others"""
    return 1.5 * normal(g, tokens, nexp) + 0.5 * normal(g, 1, nexp)


def prepare(case, seed):
    g = generator(seed)
    state = {"case": case}
    op = case["op"]
    if op == "quantize":
        n, ncol = case["rows"], case["ncol"]
        x = torch.empty((n, ncol), dtype=DTYPES[case["src"]], device=DEVICE)
        step = max(1, (1 << 27) // ncol)
        for r in range(0, n, step):              # weights with some outliers, as the benchmark's
            w = 0.02 * normal(g, min(step, n - r), ncol)
            far = torch.rand(w.shape, generator=g, device=DEVICE) < 0.001
            x[r:r + step] = torch.where(far, 0.16 * torch.sign(w), w).to(x.dtype)
        state["x"] = x
    elif op == "route":
        logits = router_logits(g, case["tokens"], case["nexp"]).to(DTYPES[case["logits"]])
        bias = 0.1 * normal(g, case["nexp"]) if case["bias"] else None
        # scores that differ by less than 32 bits resolve have no order that two ways to compute them share: a token
        # that has such among the ones it decides between is drawn again
        for _ in range(16):
            bad = (choice64(logits, bias, case)[2] < 1e-5).nonzero()[:, 0]
            if not len(bad):
                break
            logits[bad] = router_logits(g, len(bad), case["nexp"]).to(logits.dtype)
        state["logits"], state["bias"] = logits, bias
    else:
        ne1, ne0 = case["ne1"], case["ne0"]
        xtype = DTYPES[case["x"]] if case["x"] != "mxfp4" else torch.bfloat16
        names = ("w", "up") if case.get("glu") else ("w",)
        nmat = case["nexp"] if op == "experts" else 1
        state["x"] = activations(g, case["tokens"] if op == "experts" else case["m"], ne0, xtype)
        for name in names:
            state[name] = stored_blocks(g, nmat, ne1, ne0)
        if op == "experts":
            ids = router_logits(g, case["tokens"], nmat).topk(case["topk"], dim=1).indices.to(torch.int32)
            state["offsets"], state["rows"], state["slots"] = grouping(ids, nmat)
        if own:                                  # a program lays its weights out once
            gq, experts = lib()
            for name in names:
                state[name] = experts.pack(gq, state[name], nmat, ne1, ne0)
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    return run_own(state) if own else run_plain(state)


def run_own(state):
    gq, experts = lib()
    case = state["case"]
    op = case["op"]
    if op == "quantize":
        if case["form"] == "blocks":
            return experts.quantize_blocks(gq, state["x"], values=True)[1]
        return experts.quantize(gq, state["x"], values=True)[1]
    if op == "route":
        ids, weights = experts.route(gq, state["logits"], case["topk"], score=case["score"], bias=state["bias"],
                                     ngroup=case["ngroup"], keep=case["keep"], renorm=case["renorm"],
                                     scale=case["scale"])
        return [ids, weights] + list(experts.group(gq, ids, case["nexp"]))
    x = experts.quantize(gq, state["x"]) if case["x"] == "mxfp4" else state["x"]
    grouped = experts.Group(state["offsets"], state["rows"], state["slots"]) if op == "experts" else None
    return experts.matmul(gq, x, state["w"], group=grouped, up=state.get("up"), out_dtype=DTYPES[case["out"]])


def exponent_values(e):
    """2^(e - 127) in f32 of whole numbers e of 1 to 254"""
    return (e.to(torch.int32) << 23).view(torch.float32)


def plain_round(x):
    """the nearest MXFP4 values of f32 rows: blocks of 32 share 2^(floor(log2(largest)) - 2)"""
    b = x.reshape(x.shape[0], -1, 32)
    largest = b.abs().amax(dim=2, keepdim=True)
    e = torch.where(largest > 0, torch.frexp(largest).exponent + (127 - 3), 0).clamp(1, 252)
    d = exponent_values(e)
    t = b.abs() / d
    level = torch.zeros_like(t)
    for lo, hi, mid in zip(LEVELS, LEVELS[1:], MIDDLES):
        level += (hi - lo) * (t > mid)
    return (torch.sign(b) * level * d).reshape(x.shape)


def plain_weights(blocks):
    """[ne1][ne0 / 32][17] bytes -> f32 [ne1][ne0]"""
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=blocks.device)
    q = blocks[..., 1:]
    v = torch.cat((table[(q & 15).int()], table[(q >> 4).int()]), dim=-1)
    return (v * exponent_values(blocks[..., :1])).reshape(blocks.shape[0], -1)


def by_logits(case):
    return not case["bias"] and case["ngroup"] == 1


def plain_route(logits, bias, case):
    x = logits.float()
    if case["score"] == "softmax":
        p = torch.exp(x - x.amax(dim=1, keepdim=True))
        scores = p / p.sum(dim=1, keepdim=True)
    else:
        scores = 1 / (1 + torch.exp(-x))
    # both scores rise with the logits: where nothing is added to them, the logits themselves decide
    key = x if by_logits(case) else scores if bias is None else scores + bias
    if case["ngroup"] > 1:      # a group counts by the sum of its two best
        parts = key.reshape(len(x), case["ngroup"], -1)
        best = torch.sort(parts, dim=2, descending=True).values[..., :2].sum(dim=2)
        kept = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case["keep"]]
        on = torch.zeros_like(best).scatter_(1, kept, 1.0)
        key = torch.where(on[..., None] > 0, parts, -torch.inf).reshape(key.shape)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :case["topk"]]
    w = scores.gather(1, ids)
    if case["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    return ids.to(torch.int32), w * case["scale"]


def run_plain(state):
    case = state["case"]
    op = case["op"]
    if op == "quantize":
        return plain_round(state["x"].float()).to(torch.bfloat16)
    if op == "route":
        ids, weights = plain_route(state["logits"], state["bias"], case)
        return [ids, weights] + list(grouping(ids, case["nexp"]))
    x = plain_round(state["x"].float()) if case["x"] == "mxfp4" else state["x"].float()
    if op == "matmul":
        return (x @ plain_weights(state["w"][0]).T).to(DTYPES[case["out"]])
    out = torch.empty((len(state["rows"]), case["ne1"]), dtype=DTYPES[case["out"]], device=x.device)
    offsets = state["offsets"].tolist()
    for e in range(case["nexp"]):
        a, b = offsets[e], offsets[e + 1]
        if a == b:
            continue
        xe = x[state["rows"][a:b].long()]
        y = xe @ plain_weights(state["w"][e]).T
        if case["glu"]:
            y = y / (1 + torch.exp(-y)) * (xe @ plain_weights(state["up"][e]).T)
        out[a:b] = y.to(out.dtype)
    return out


# ---------------------------------------------------------------- the definition in 64 bits
def round64(x):
    middles = torch.tensor(MIDDLES, dtype=torch.float64, device=x.device)
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    step = max(1, (1 << 25) // x.shape[1])
    for r in range(0, len(x), step):
        v = x[r:r + step].double().reshape(-1, 32)
        top = v.abs().max(dim=1, keepdim=True).values
        unit = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2)
        near = levels[torch.bucketize((v / unit).abs(), middles)]         # (a tie goes to the smaller)
        out[r:r + step] = torch.copysign(near * unit, v).reshape(-1, x.shape[1])
    return out


def weights64(blocks):
    q = blocks[..., 1:].int()
    code = torch.stack((q & 15, q >> 4), dim=-2).flatten(-2)
    size = code & 7
    m, e = (size & 1).double(), size >> 1
    v = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2((e - 1).double()))
    v = torch.where(code >= 8, -v, v) * torch.exp2(blocks[..., :1].double() - 127)
    return v.flatten(-2)


def choice64(logits, bias, case):
    """ids, weights and the smallest gap between different scores that the choice rests on"""
    x = logits.double()
    score = torch.softmax(x, dim=1) if case["score"] == "softmax" else torch.sigmoid(x)
    key = x if by_logits(case) else score if bias is None else score + bias.double()
    gap = torch.full((len(x),), torch.inf, dtype=torch.float64, device=x.device)

    def closest(sorted_keys):
        d = sorted_keys[:, :-1] - sorted_keys[:, 1:]
        return torch.where(d > 0, d, torch.inf).amin(dim=1) if d.shape[1] else gap
    if case["ngroup"] > 1:
        parts = key.unflatten(1, (case["ngroup"], -1))
        best = parts.topk(min(2, parts.shape[2]), dim=2).values.sum(dim=2)
        by, order = torch.sort(best, dim=1, descending=True, stable=True)
        if case["keep"] < case["ngroup"]:
            gap = torch.minimum(gap, closest(by[:, case["keep"] - 1:case["keep"] + 1]))
        out = torch.ones_like(best, dtype=torch.bool).scatter(1, order[:, :case["keep"]], False)
        key = parts.masked_fill(out[..., None], -torch.inf).flatten(1)
    by, order = torch.sort(key, dim=1, descending=True, stable=True)
    if not by_logits(case):
        gap = torch.minimum(gap, closest(by[:, :case["topk"] + 1]))
    ids = order[:, :case["topk"]]
    w = torch.take_along_dim(score, ids, dim=1)
    if case["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    return ids.to(torch.int32), w * case["scale"], gap


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "quantize":
        return round64(state["x"])
    if op == "route":
        ids, weights, _ = choice64(state["logits"], state["bias"], case)
        return [ids, weights] + list(grouping(ids, case["nexp"]))
    x = round64(state["x"]) if case["x"] == "mxfp4" else state["x"].double()
    if op == "matmul":
        return x @ weights64(state["w"][0]).T
    out = torch.empty((len(state["rows"]), case["ne1"]), dtype=torch.float64, device=x.device)
    offsets = state["offsets"].tolist()
    for e in range(case["nexp"]):
        a, b = offsets[e], offsets[e + 1]
        if a == b:
            continue
        rows = x.index_select(0, state["rows"][a:b].long())
        y = rows @ weights64(state["w"][e]).T
        if case["glu"]:
            y = y * torch.sigmoid(y) * (rows @ weights64(state["up"][e]).T)
        out[a:b] = y
    return out

"""Cases of the operators that score rows held in 8-bit integers and pick the best continuations: quantization of rows
to int8 with a scale each, the int8 product with scales for rows and columns, the same product for rows that arrive in
floating point, and the selection over the beams of a group with the reordering of what the beams carry.

`run` computes a pass either in elementary torch operations (`own` false) or through needle_amd (`own` true).
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_contexts = {}


def listed():
    return [
        # one query embedding on its way into an int8 scan: the smallest call, latency alone
        dict(name="quantize_one_query", op="quantize", rows=1, dim=768, pad=0, value="f32"),
        # a base of embeddings held in int8 from here on, an odd number of rows
        dict(name="quantize_base", op="quantize", rows=200_003, dim=384, pad=0, value="f32"),
        # one query against a million rows: the product is a stream over the int8 base
        dict(name="scores_one_query", op="matmul", m=1, n=1_000_000, k=384, pad=0, bias=False, out="f32"),
        # a thousand queries against 100K rows of 128 dimensions: the scores are what moves
        dict(name="scores_batch", op="matmul", m=1000, n=100_000, k=128, pad=0, bias=False, out="f32"),
        # a Matryoshka prefix of odd length out of longer rows, few queries, sizes that fill no tile
        dict(name="scores_prefix", op="matmul", m=37, n=50_001, k=301, pad=83, bias=False, out="f32"),
        # a large product of a model's layer, compute bound
        dict(name="product_large", op="matmul", m=8192, n=8192, k=4096, pad=0, bias=False, out="bf16"),
        # the last layer at one position of four beams: the int8 table of a vocabulary is streamed
        dict(name="linear_one_position", op="linear", m=4, n=32_000, k=1024, pad=0, bias=False, value="bf16", out="f32"),
        # a layer over a whole prompt, with a bias
        dict(name="linear_prompt", op="linear", m=4096, n=8192, k=2048, pad=0, bias=True, value="bf16", out="bf16"),
        # one request, four beams: latency
        dict(name="beam_one_request", op="beam", groups=1, beams=4, vocab=32_000, k=4, value="f32", normalize=True,
             first=False, mask=0.0, finished=False, state="none", heads=0, room=0, length=0),
        # many requests with the keys and values of their beams: states move with the picks
        dict(name="beam_many_requests", op="beam", groups=64, beams=8, vocab=131_072, k=8, value="bf16", normalize=True,
             first=False, mask=0.0, finished=False, state="cache", heads=8, room=512, length=384),
        # continuations that a constraint admits (1 % of the tokens, for some beams none), some beams ended
        dict(name="beam_constrained", op="beam", groups=16, beams=5, vocab=50_021, k=10, value="f16", normalize=True,
             first=False, mask=0.01, finished=True, state="none", heads=0, room=0, length=0),
        # a hop of a retrieval chain: scores of base rows as they are, the chains' query vectors move with the picks
        dict(name="beam_hop", op="beam", groups=32, beams=10, vocab=100_003, k=64, value="f32", normalize=False,
             first=False, mask=0.0, finished=False, state="vectors", heads=1, room=384, length=384),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "matmul", "linear", "beam", "beam"])
    if op == "quantize":
        dim = _log(rng, 8, 4096)
        return dict(op=op, rows=_log(rng, 1, min(200_000, 76_000_000 // dim)), dim=dim, pad=rng.choice([0, 0, 1, 16, 37]),
                    value=rng.choice(["f32", "f16", "bf16"]))
    if op in ("matmul", "linear"):
        k = _log(rng, 16, 4096)
        m = _log(rng, 1, 8192)
        n = _log(rng, 16, min(1_000_000, 300_000_000 // k, 80_000_000 // m))
        c = dict(op=op, m=m, n=n, k=k, pad=rng.choice([0, 0, 0, 16, 5]), bias=rng.random() < 0.4, out=rng.choice(["f32", "f32", "bf16", "f16"]))
        return c if op == "matmul" else dict(c, value=rng.choice(["f32", "f16", "bf16"]))
    beams, groups = _log(rng, 1, 16), _log(rng, 1, 64)
    vocab = _log(rng, 1000, min(131_072, 60_000_000 // (beams * groups)))
    state = rng.choice(["none", "cache", "vectors"])
    finished = rng.random() < 0.3
    first = state != "none" and not finished and rng.random() < 0.3
    mask = rng.choice([0.0, 0.01, 0.3]) if state == "none" else 0.0
    # chains that move with the picks need a pick for every place: ended beams then get no more places than beams
    k = beams if finished and state != "none" else _log(rng, 1, 64)
    heads, room = rng.choice([2, 4, 8]), _log(rng, 8, 400)
    if state == "cache":
        room = max(1, min(room, 400_000 // (groups * max(k, beams))))
    length = rng.randint(1, room)
    if state == "vectors":
        heads, room = 1, _log(rng, 8, 1536)
        length = room
    return dict(op=op, groups=groups, beams=beams, vocab=vocab, k=k, value=rng.choice(["f32", "f16", "bf16"]),
                normalize=rng.random() < 0.7, first=first, mask=mask, finished=finished, state=state, heads=heads, room=room, length=length)


# ---- inputs ------------------------------------------------------------------------------------------


def _codes(x):
    """Rows as int8 codes with a scale each: scale = max |x| / 127 in 32 bits, code = the whole number nearest to
    x / scale (half to even).  The quotient is formed in 64 bits: in 32 it can round onto a half that it is not."""
    x = x.float()
    scale = (x.abs().amax(dim=1) / 127.0)
    codes = torch.round(x.double() / torch.where(scale > 0, scale, torch.ones_like(scale)).double()[:, None])
    return codes.clamp_(-127, 127).to(torch.int8), scale


def _vectors(g, rows, dim, pad, value):
    """Embeddings: normal components, a few of them large in every row; a row of zeros now and then."""
    x = torch.randn(rows, dim + pad, generator=g, device="cuda")
    x[:, :: max(dim // 4, 1)] *= 4.0
    x *= torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))
    if rows > 8:
        x[rows // 2] = 0.0
    return x.to(TYPES[value])[:, :dim]


def _table(g, rows, dim, pad):
    """Codes [rows, dim] of a wider int8 table, with their scales."""
    codes = torch.randn(rows, dim + pad, generator=g, device="cuda", dtype=torch.bfloat16).mul_(40.0).clamp_(-127, 127).to(torch.int8)
    return codes[:, :dim], torch.rand(rows, generator=g, device="cuda") * 0.01 + 1e-4


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    if case["op"] == "quantize":
        s["x"] = _vectors(g, case["rows"], case["dim"], case["pad"], case["value"])
        s["codes"] = torch.empty(case["rows"], case["dim"], dtype=torch.int8, device="cuda")
        s["scales"] = torch.empty(case["rows"], device="cuda")
        return s
    if case["op"] in ("matmul", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        s["b"], s["b_scales"] = _table(g, n, k, case["pad"])
        if case["op"] == "matmul":
            s["a"], s["a_scales"] = _table(g, m, k, case["pad"])
        else:
            s["x"] = _vectors(g, m, k, case["pad"], case["value"])
        s["bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        s["out"] = torch.empty(m, n, dtype=TYPES[case["out"]], device="cuda")
        return s
    rows, picks, v = case["groups"] * case["beams"], case["groups"] * case["k"], case["vocab"]
    s["logits"] = (torch.randn(rows, v, generator=g, device="cuda") * 2.5).to(TYPES[case["value"]])
    scores = -torch.rand(case["groups"], case["beams"], generator=g, device="cuda") * 4.0 - 10.0
    if case["first"]:  # nothing is chosen yet: one beam of every group is alive
        scores[:, 0], scores[:, 1:] = 0.0, -math.inf
    s["scores"] = scores.reshape(-1)
    s["mask"] = s["finished"] = None
    if case["mask"]:
        bits = torch.rand(rows, -(-v // 32), 32, generator=g, device="cuda") < case["mask"]
        bits[1::7] = False  # beams that no continuation is admitted for
        s["mask"] = (bits.long() << torch.arange(32, device="cuda")).sum(dim=2).to(torch.int32)
    if case["finished"]:
        s["finished"] = torch.rand(rows, generator=g, device="cuda") < 0.25
    s["states"] = []
    if case["state"] == "cache":
        shape = (case["heads"], case["room"], 64)
        s["states"] = [tuple(torch.randn((r,) + shape, generator=g, device="cuda", dtype=torch.bfloat16)[:, :, : case["length"]]
                             for r in (rows, picks)) for _ in range(2)]
    elif case["state"] == "vectors":
        s["states"] = [(torch.randn(rows, case["room"], generator=g, device="cuda"), torch.empty(picks, case["room"], device="cuda")),
                       (torch.randint(0, v, (rows, 5), generator=g, device="cuda", dtype=torch.int32),
                        torch.empty(picks, 5, device="cuda", dtype=torch.int32))]
    for name, dtype in (("parents", torch.int32), ("tokens", torch.int32), ("picked", torch.float32)):
        s[name] = torch.empty(case["groups"], case["k"], dtype=dtype, device="cuda")
    s["counts"] = torch.empty(case["groups"], dtype=torch.int32, device="cuda")
    return s


# ---- one pass ------------------------------------------------------------------------------------------


def _context():
    if "ctx" not in _contexts:
        import needle_amd

        _contexts["ctx"] = needle_amd.Context(torch.cuda.current_device())
    return _contexts["ctx"]


def _product(a, a_scales, s):
    y = (a.float() @ s["b"].float().T) * a_scales[:, None] * s["b_scales"][None, :]
    if s["bias"] is not None:
        y = y + s["bias"][None, :]
    return y.to(TYPES[s["case"]["out"]])


END = 2  # the token that an ended beam repeats


def _beam(s):
    c = s["case"]
    groups, beams, v, k = c["groups"], c["beams"], c["vocab"], c["k"]
    x = s["logits"].float()
    token = torch.arange(v, device="cuda")
    if s["mask"] is not None:
        x = torch.where((s["mask"][:, token >> 5] >> (token & 31)) & 1 != 0, x, -math.inf)
    wide = x.double()
    # the order of one beam's tokens: by logit, then the lowest token, as one whole number
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() * 2**32 + (v - 1 - token)
    nothing = -(2**63)
    order = torch.where(x.isnan() | (x == -math.inf), torch.full_like(order, nothing), order)
    best = min(k, v)
    top = torch.topk(order, best, dim=1).values
    picked = torch.where(top == nothing, torch.zeros_like(top), v - 1 - (top & 0xFFFFFFFF))
    total = torch.gather(wide, 1, picked)
    if c["normalize"]:  # differences of totals decide between beams: 64 bits
        most = wide.amax(dim=1, keepdim=True)
        total = total - (most + torch.log(torch.exp(wide - most).sum(dim=1, keepdim=True)))
    total = s["scores"].double()[:, None] + total
    total = torch.where((top == nothing) | total.isnan(), -math.inf, total)
    if s["finished"] is not None:  # an ended beam offers its own score with the end token, and nothing else
        ended = s["finished"][:, None]
        only = torch.arange(best, device="cuda")[None, :] == 0
        total = torch.where(ended, torch.where(only, s["scores"].double()[:, None], -math.inf), total)
        picked = torch.where(ended, torch.full_like(picked, END), picked)
    total, at = torch.sort(total.view(groups, beams * best), dim=1, descending=True, stable=True)
    total, at = total[:, :k], at[:, :k]
    if at.shape[1] < k:
        more = k - at.shape[1]
        total = torch.nn.functional.pad(total, (0, more), value=-math.inf)
        at = torch.nn.functional.pad(at, (0, more))
    there = total != -math.inf
    parents = torch.where(there, at // best, -1).to(torch.int32)
    tokens = torch.where(there, torch.gather(picked.view(groups, beams * best), 1, at), -1).to(torch.int32)
    # in the cases with states every group fills its k places
    rows = (torch.arange(groups, device="cuda")[:, None] * beams + at // best).reshape(-1)
    return dict(parents=parents, tokens=tokens, scores=total.float(), counts=there.sum(dim=1).to(torch.int32),
                states=[src.index_select(0, rows) for src, _ in s["states"]])


def run(state):
    s, c = state, state["case"]
    if own:
        ctx = _context()
        if c["op"] == "quantize":
            ctx.quantize_rows_device(s["x"], s["codes"], s["scales"])
            return dict(codes=s["codes"], scales=s["scales"])
        if c["op"] == "matmul":
            ctx.matmul_i8_device(s["a"], s["a_scales"], s["b"], s["b_scales"], s["out"], d_bias=s["bias"])
            return dict(out=s["out"])
        if c["op"] == "linear":
            ctx.linear_i8_device(s["x"], s["b"], s["b_scales"], s["out"], d_bias=s["bias"])
            return dict(out=s["out"])
        ctx.beam_select_device(s["logits"], s["scores"], c["k"], s["parents"], s["tokens"], s["picked"], s["counts"],
                               beams=c["beams"], normalize=c["normalize"], d_mask=s["mask"], d_finished=s["finished"],
                               end_token=END, states=s["states"])
        return dict(parents=s["parents"], tokens=s["tokens"], scores=s["picked"], counts=s["counts"],
                    states=[dst for _, dst in s["states"]])
    if c["op"] == "quantize":
        codes, scales = _codes(s["x"])
        return dict(codes=codes, scales=scales)
    if c["op"] == "matmul":
        return dict(out=_product(s["a"], s["a_scales"], s))
    if c["op"] == "linear":
        return dict(out=_product(*_codes(s["x"]), s))
    return _beam(s)


# ---- what a pass cannot do without ---------------------------------------------------------------------


def work(case):
    if case["op"] == "quantize":
        n = case["rows"] * case["dim"]
        return {"bytes": n * (SIZE[case["value"]] + 1) + 4 * case["rows"], "flops": 2 * n}
    if case["op"] in ("matmul", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        a = m * k + 4 * m if case["op"] == "matmul" else m * k * SIZE[case["value"]]
        return {"bytes": a + n * k + 4 * n * (2 if case["bias"] else 1) + m * n * SIZE[case["out"]], "flops": 2 * m * n * k}
    rows, picks = case["groups"] * case["beams"], case["groups"] * case["k"]
    moved = rows * case["vocab"] * SIZE[case["value"]] + 4 * rows + 12 * picks
    if case["mask"]:
        moved += rows * -(-case["vocab"] // 32) * 4
    if case["state"] == "cache":
        moved += 2 * (rows + picks) * case["heads"] * case["length"] * 64 * 2
    elif case["state"] == "vectors":
        moved += (rows + picks) * (case["room"] + 5) * 4
    return {"bytes": moved, "flops": (3 if case["normalize"] else 1) * rows * case["vocab"]}


# ---- the definitions in 64 bits -------------------------------------------------------------------------


def _exact_codes(x):
    x = x.double().cpu().numpy()
    scale = (np.abs(x).max(axis=1) / 127.0).astype(np.float32).astype(np.float64)
    return np.clip(np.rint(np.divide(x, scale[:, None], out=np.zeros_like(x), where=scale[:, None] > 0)), -127, 127), scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        x = s["x"].double().cpu().numpy()
        return dict(codes=_exact_codes(s["x"])[0].astype(np.int8), scales=np.abs(x).max(axis=1) / 127.0)
    if case["op"] in ("matmul", "linear"):
        a, a_scales = (s["a"].double(), s["a_scales"].double()) if case["op"] == "matmul" else \
            (torch.from_numpy(v).cuda() for v in _exact_codes(s["x"]))
        out = torch.matmul(a, s["b"].double().t().contiguous())
        out.mul_(a_scales.unsqueeze(1)).mul_(s["b_scales"].double().unsqueeze(0))
        if s["bias"] is not None:
            out.add_(s["bias"].double())
        return dict(out=out)
    groups, beams, v, k = case["groups"], case["beams"], case["vocab"], case["k"]
    scores = np.full((groups, k), -np.inf)
    start = s["scores"].double().cpu().numpy()
    ended = np.zeros(groups * beams, dtype=bool) if s["finished"] is None else s["finished"].cpu().numpy()
    for i in range(groups):
        offers = []
        for r in range(i * beams, (i + 1) * beams):
            if ended[r]:
                offers.append(np.array([start[r]]))
                continue
            x = s["logits"][r].double().cpu().numpy()
            if s["mask"] is not None:
                words = s["mask"][r].cpu().numpy().view(np.uint8)
                x = x[np.unpackbits(words, bitorder="little")[:v].astype(bool)]
            if x.size == 0:
                continue
            if case["normalize"]:
                x = x - (x.max() + math.log(np.exp(x - x.max()).sum()))
            offers.append(start[r] + np.partition(x, max(x.size - k, 0))[max(x.size - k, 0):])
        best = np.sort(np.concatenate(offers))[::-1][:k] if offers else np.zeros(0)
        scores[i, : best.size] = best
    return dict(parents=None, tokens=None, scores=scores, counts=(scores > -np.inf).sum(axis=1).astype(np.int32),
                states=[None for _ in s["states"]])

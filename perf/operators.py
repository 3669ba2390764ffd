"""The operators of a beam-search decode step, as cases that can be timed.

Four kinds of pass:

  norm     the sum after a block and the next block's norm: the block's output,
           normalized or not, times its gate, onto the scaled residual, and the
           rmsnorm of that sum
  linear   a product of 4-bit microscaled operands: bf16 activations quantized
           to MXFP4, then multiplied with MXFP4 weights
  select   beam search's choice among beams x vocabulary
  reorder  the beams' states (token histories, caches) following their parents

Where `own` is false a pass is computed with elementary torch operations,
where it is true with the framework's entry points.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EPS = 1e-5
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # magnitudes of the 4-bit codes
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}


def _l2c():
    path = os.path.join(ROOT, "cuda-elastic_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import l2c
    return l2c


# ---------------------------------------------------------------------------
# Cases.

def _norm(batch, size, residual, block, normalized, post, gate, name=None):
    c = {"kind": "norm", "batch": batch, "size": size, "residual": residual, "block": block, "normalized": normalized,
         "post": post, "gate": gate}
    return dict(c, name=name) if name else c


def _linear(batch, size, rows, name=None):
    c = {"kind": "linear", "batch": batch, "size": size, "rows": rows}
    return dict(c, name=name) if name else c


def _select(batch, beams, vocab, name=None):
    c = {"kind": "select", "batch": batch, "beams": beams, "vocab": vocab}
    return dict(c, name=name) if name else c


def _reorder(element, groups, batch, beams, pieces, positions, live, width, name=None):
    c = {"kind": "reorder", "element": element, "groups": groups, "batch": batch, "beams": beams, "pieces": pieces,
         "positions": positions, "live": live, "width": width}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One decoded token between two blocks: nothing but latency.
        _norm(1, 4096, "f32", "f32", "bf16", True, "one", "norm_1x4096"),
        # A ragged batch with a bf16 residual stream and a gate for every token.
        _norm(130, 5003, "bf16", "bf16", "bf16", False, "row", "norm_130x5003"),
        # The largest profiled batch, an fp32 stream whose norm goes into a bf16 product.
        _norm(1024, 16384, "f32", "f32", "bf16", True, "one", "norm_1024x16384"),
        # One token through a 4096-wide layer: the weights streamed once.
        _linear(1, 4096, 11008, "linear_1x4096x11008"),
        # A ragged decode batch whose length is no multiple of 64.
        _linear(40, 5024, 8004, "linear_40x5024x8004"),
        # A prefill chunk, or a full decode batch.
        _linear(256, 4096, 11008, "linear_256x4096x11008"),
        # The largest profiled shape.
        _linear(1024, 16384, 8192, "linear_1024x16384x8192"),
        # One request with four beams.
        _select(1, 4, 32000, "select_1x4x32000"),
        # A few requests with many beams over a large vocabulary.
        _select(8, 16, 131072, "select_8x16x131072"),
        # A full batch of requests, rows of no multiple of four logits.
        _select(256, 4, 32003, "select_256x4x32003"),
        # The token histories of a few requests, one of which follows each step.
        _reorder("int32", 1, 8, 4, 1, 256, 100, 1, "reorder_history_8x4x100"),
        # Keys and values of four layers: eight heads, three quarters full.
        _reorder("bf16", 8, 8, 8, 8, 512, 384, 128, "reorder_cache_8x8x8x8x384x128"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("norm", "linear", "linear", "select", "select", "reorder"))
    granule = 256 if rng.random() < 0.4 else 1  # four sizes in ten are a model's
    if kind == "norm":
        size = max(granule, round(_log_int(rng, 288, 16384) / granule) * granule)
        return _norm(_log_int(rng, 1, 1024), size, rng.choice(("f32", "bf16")), rng.choice(("f32", "bf16")),
                     rng.choice(("f32", "bf16")), rng.random() < 0.5, rng.choice(("none", "one", "row", "sixteen")))
    if kind == "linear":
        granule = max(granule, 32)
        batch, size, rows = _log_int(rng, 1, 1024), _log_int(rng, 288, 16384), _log_int(rng, 288, 11008)
        size = max(granule, round(size / granule) * granule)
        while batch * size * rows > 1024 * 16384 * 8192:
            batch //= 2
        return _linear(batch, size, rows)
    if kind == "select":
        batch, beams = _log_int(rng, 1, 256), rng.randint(1, 32)
        vocab = max(granule, round(_log_int(rng, 288, 131072) / granule) * granule)
        while batch * beams * vocab > 256 * 4 * 32003:
            if batch > 1:
                batch //= 2
            else:
                beams //= 2
        return _select(batch, beams, vocab)
    batch, beams = _log_int(rng, 1, 64), rng.randint(2, 16)
    if rng.random() < 0.4:
        positions = _log_int(rng, 16, 4096)
        return _reorder("int32", 1, batch, beams, 1, positions, rng.randint(1, positions), 1)
    groups, pieces = 2 * rng.randint(1, 8), rng.choice((1, 2, 4, 8, 5))
    width, positions = rng.choice((64, 80, 128, 13)), _log_int(rng, 16, 1024)
    while groups * batch * beams * pieces * positions * width > 8 * 8 * 8 * 8 * 384 * 128:
        if batch > 1:
            batch //= 2
        else:
            positions //= 2
    return _reorder("bf16", groups, batch, beams, pieces, positions, rng.randint(1, positions), width)


# ---------------------------------------------------------------------------
# Inputs, from the seed alone.

def _normal(gen, *shape):
    return torch.empty(*shape, device="cuda").normal_(generator=gen)


def _gate_rows(c):
    """(rows of gates, rows of the batch that share one)."""
    per = {"none": 1, "one": c["batch"], "row": 1, "sixteen": 16}[c["gate"]]
    return (0 if c["gate"] == "none" else -(-c["batch"] // per)), per


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    c = dict(case)
    uniform = lambda *s: torch.empty(*s, device="cuda").uniform_(0.5, 1.5, generator=gen)  # noqa: E731
    if c["kind"] == "norm":
        rows, per = _gate_rows(c)
        c.update(
            per=per, x=(2.0 * _normal(gen, c["batch"], c["size"])).to(TYPES[c["residual"]]),
            y=_normal(gen, c["batch"], c["size"]).to(TYPES[c["block"]]),
            w=uniform(c["size"]), pw=uniform(c["size"]) if c["post"] else None,
            g=0.5 * _normal(gen, rows, c["size"]) if rows else None, scale=0.75,
            h=torch.empty(c["batch"], c["size"], device="cuda", dtype=TYPES[c["residual"]]),
            n=torch.empty(c["batch"], c["size"], device="cuda", dtype=TYPES[c["normalized"]]))
    elif c["kind"] == "linear":
        x = _normal(gen, c["batch"], c["size"])
        x[:, torch.randint(c["size"], (4,), generator=gen, device="cuda")] *= 20.0  # outlier channels
        codes, scales = _to_mxfp4(_normal(gen, c["rows"], c["size"]) / math.sqrt(c["size"]))
        c.update(x=x.bfloat16(), wc=codes, ws=scales,
                 xc=torch.empty(c["batch"], c["size"] // 2, device="cuda", dtype=torch.uint8),
                 xs=torch.empty(c["batch"], c["size"] // 32, device="cuda", dtype=torch.uint8),
                 out=torch.empty(c["batch"], c["rows"], device="cuda"))
    elif c["kind"] == "select":
        n, vocab = c["batch"] * c["beams"], c["vocab"]
        # The beams of a request lie within a few units of each other; about one in twelve has ended.
        scores = -20.0 - 2.0 * _normal(gen, n).abs()
        tokens = torch.randint(3, vocab, (n,), generator=gen, device="cuda", dtype=torch.int32)
        tokens[torch.rand(n, generator=gen, device="cuda") < 0.08] = 2
        c.update(eos=2, logits=3.0 * _normal(gen, n, vocab), scores=scores, tokens=tokens, steps=64, step=17,
                 scores_out=torch.empty(n, device="cuda"), tokens_out=torch.empty(n, device="cuda", dtype=torch.int32),
                 parents=torch.empty(n, device="cuda", dtype=torch.int32),
                 generated=torch.zeros(n, 64, device="cuda", dtype=torch.int32))
        # At most this by the formula that the entry point documents.
        c["workspace"] = torch.empty(n * -(-vocab // 1024) * (8 * c["beams"] + 16), device="cuda", dtype=torch.uint8)
    else:
        shape = (c["groups"], c["batch"], c["beams"], c["pieces"], c["positions"], c["width"])
        if c["element"] == "int32":
            state = torch.randint(32000, shape, generator=gen, device="cuda", dtype=torch.int32)
        else:
            state = torch.empty(shape, device="cuda", dtype=torch.bfloat16).normal_(generator=gen)
        parents = torch.randint(c["beams"], (c["batch"], c["beams"]), generator=gen, device="cuda", dtype=torch.int32)
        parents[torch.rand(parents.shape, generator=gen, device="cuda") < 0.02] = -1  # beams without a successor
        c.update(state=state, out=torch.zeros_like(state), parents=parents)
    return c


# ---------------------------------------------------------------------------
# The plain forms.

def _pow2(exponent):
    return ((exponent + 127).clamp(1, 254).int() << 23).view(torch.float32)


def _to_mxfp4(x):
    """(codes, two a byte; scale bytes) of rows of 32-value blocks: the block's exponent is
    floor(log2(maximum)) - 2, the codes the nearest of x * 2^-exponent, ties to the even code."""
    blocks = x.float().reshape(x.shape[0], -1, 32)
    exponent = (torch.frexp(blocks.abs().amax(-1)).exponent - 3).clamp(-127, 127)
    exponent = torch.where(blocks.abs().amax(-1) > 0, exponent, torch.full_like(exponent, -127))
    v = blocks * _pow2(-exponent).unsqueeze(-1)
    a = v.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte()
            + (a >= 3.5).byte() + (a > 5.0).byte())
    code = (code + 8 * ((v < 0) & (code > 0)).byte()).reshape(x.shape[0], -1, 2)
    return code[..., 0] + 16 * code[..., 1], (exponent + 127).to(torch.uint8)


def _of_mxfp4(codes, scales):
    values = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    v = torch.stack((values[(codes & 15).int()], values[(codes >> 4).int()]), -1).reshape(*scales.shape, 32)
    return (v * _pow2(scales.int() - 127).unsqueeze(-1)).reshape(codes.shape[0], -1)


def _plain_norm(s):
    x, z = s["x"].float(), s["y"].float()
    if s["pw"] is not None:
        z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS) * s["pw"]
    if s["g"] is not None:
        z = z * s["g"].repeat_interleave(s["per"], 0)[:s["batch"]]
    h = s["scale"] * x + z
    n = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["w"]
    return {"residual": h.to(s["h"].dtype), "normalized": n.to(s["n"].dtype)}


def _plain_linear(s):
    return _of_mxfp4(*_to_mxfp4(s["x"])) @ _of_mxfp4(s["wc"], s["ws"]).t()


def _plain_select(s):
    """In 64 bits: what matters is the order of scores that may lie next to each other."""
    batch, beams, vocab = s["batch"], s["beams"], s["vocab"]
    l = s["logits"].double()
    top = l.amax(-1, keepdim=True)
    score = s["scores"].double().unsqueeze(-1) + (l - top - (l - top).exp().sum(-1, keepdim=True).log())
    ended = (s["tokens"] == s["eos"]).unsqueeze(-1)
    last = torch.arange(vocab, device=l.device) == s["eos"]
    score = torch.where(ended, torch.where(last, s["scores"].double().unsqueeze(-1), -math.inf), score)
    best, at = torch.sort(score.reshape(batch, beams * vocab), dim=-1, descending=True, stable=True)
    best, at = best[:, :beams].reshape(-1), at[:, :beams].reshape(-1)
    parents = torch.where(best > -math.inf, at // vocab, -1).int()
    tokens = torch.where(best > -math.inf, at % vocab, -1).int()
    s["generated"][:, s["step"]] = tokens
    return {"scores": best.float(), "tokens": tokens, "parents": parents, "generated": s["generated"]}


def _plain_reorder(s):
    live, parents = s["live"], s["parents"].long()
    rows = torch.arange(s["batch"], device=parents.device).unsqueeze(-1)
    moved = s["state"][:, rows, parents.clamp(min=0)][..., :live, :]
    keep = (parents < 0).reshape(1, s["batch"], s["beams"], 1, 1, 1)
    s["out"][..., :live, :] = torch.where(keep, s["out"][..., :live, :], moved)
    return s["out"]


def run(s):
    kind = s["kind"]
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "select": _plain_select, "reorder": _plain_reorder}[kind](s)
    l2c = _l2c()
    if kind == "norm":
        l2c.residual_rmsnorm(s["n"], s["h"], s["x"], s["y"], s["w"], s["size"], s["batch"], block_weight=s["pw"],
                             gate=s["g"], rows_per_gate=s["per"], residual_scale=s["scale"], eps=EPS)
        return {"residual": s["h"], "normalized": s["n"]}
    if kind == "linear":
        l2c.quantize_mxfp4_bf16(s["xc"], s["xs"], s["x"], s["batch"], s["size"])
        l2c.matmul_mxfp4(s["out"], s["xc"], s["xs"], s["wc"], s["ws"], s["batch"], s["size"], s["rows"])
        return s["out"]
    if kind == "select":
        l2c.decoder_beam_select(s["scores_out"], s["tokens_out"], s["parents"], s["generated"], s["logits"],
                                s["scores"], s["tokens"], s["eos"], s["vocab"], s["beams"], s["batch"], s["steps"],
                                s["step"], s["workspace"])
        return {"scores": s["scores_out"], "tokens": s["tokens_out"], "parents": s["parents"],
                "generated": s["generated"]}
    unit = s["width"] * s["state"].element_size()
    piece = s["positions"] * unit
    row = s["pieces"] * piece
    l2c.decoder_beam_reorder(s["out"], s["state"], s["parents"], s["beams"], s["batch"], s["live"] * unit,
                             row_stride=row, pieces=s["pieces"], piece_stride=piece, groups=s["groups"],
                             group_stride=s["batch"] * s["beams"] * row)
    return s["out"]


# ---------------------------------------------------------------------------
# What a pass cannot do without.

def work(case):
    c = case
    if c["kind"] == "norm":
        n = c["batch"] * c["size"]
        rows, _ = _gate_rows(c)
        each = 2 * BYTES[c["residual"]] + BYTES[c["block"]] + BYTES[c["normalized"]]
        return {"bytes": n * each + 4 * c["size"] * (1 + c["post"] + rows), "flops": n * (8 + 4 * c["post"])}
    if c["kind"] == "linear":
        b, k, r = c["batch"], c["size"], c["rows"]
        return {"bytes": 2 * b * k + r * (k // 2 + k // 32) + 4 * b * r, "flops": 2 * b * k * r}
    if c["kind"] == "select":
        n = c["batch"] * c["beams"]
        return {"bytes": 4 * n * c["vocab"] + 24 * n, "flops": 5 * n * c["vocab"]}
    rows = c["groups"] * c["batch"] * c["beams"]
    piece = c["pieces"] * c["live"] * c["width"] * (4 if c["element"] == "int32" else 2)
    wanted = 1.0 - (1.0 - 1.0 / c["beams"]) ** c["beams"]  # of the rows, by the parents that prepare() draws
    return {"bytes": int(rows * piece * (1.0 + wanted)) + 4 * c["batch"] * c["beams"], "flops": 0}


# ---------------------------------------------------------------------------
# The operators in 64 bits, from their definitions.

def exact(case, seed):
    if case["kind"] == "reorder":
        return None  # copies
    s = prepare(case, seed)

    def norm():
        def normed(v, w):
            return v / torch.sqrt(torch.linalg.vector_norm(v, dim=1, keepdim=True) ** 2 / s["size"] + EPS) * w.double()

        z = s["y"].double()
        if s["post"]:
            z = normed(z, s["pw"])
        for r in range(s["batch"] if s["g"] is not None else 0):
            z[r] *= s["g"][r // s["per"]].double()
        h = z + s["x"].double() * s["scale"]
        return {"residual": h, "normalized": normed(h, s["w"])}

    def linear():
        x = s["x"].double().reshape(s["batch"], -1, 32)
        # The exponent field of the largest of a block's bf16 patterns.
        field = ((s["x"].view(torch.int16).int() & 0x7fff) >> 7).reshape(s["batch"], -1, 32).amax(-1, keepdim=True)
        scale = torch.pow(2.0, (field - 129).clamp(min=-127).double())
        grid = torch.tensor(GRID, device=x.device, dtype=torch.float64)
        even_first = 1e-9 * (torch.arange(8, device=x.device) % 2)
        q = torch.empty_like(x)
        for r in range(0, s["batch"], 64):  # a few rows at a time: eight distances a value
            away = ((x[r:r + 64] / scale[r:r + 64]).abs().unsqueeze(-1) - grid).abs() + even_first
            q[r:r + 64] = grid[away.argmin(-1)] * x[r:r + 64].sign() * scale[r:r + 64]
        w = torch.empty(s["rows"], s["size"], device=x.device, dtype=torch.float64)
        for half in (0, 1):
            code = (s["wc"].int() >> (4 * half)) & 15
            e, m = (code >> 1) & 3, (code & 1).double()
            magnitude = torch.where(e == 0, m / 2, (1 + m / 2) * torch.pow(2.0, e.double() - 1))
            w[:, half::2] = torch.where(code > 7, -magnitude, magnitude)
        w *= torch.pow(2.0, s["ws"].double() - 127).repeat_interleave(32, 1)
        return q.reshape(s["batch"], -1) @ w.t()

    def select():  # each beam's own best, then the best of its request's
        most = min(s["beams"], s["vocab"])
        logits = s["logits"].double()
        own_best = torch.topk(logits, most).values - torch.logsumexp(logits, 1, keepdim=True)
        ended = torch.full_like(own_best, -math.inf)
        ended[:, 0] = 0.0
        own_best = torch.where((s["tokens"] == s["eos"]).unsqueeze(1), ended, own_best) + s["scores"].double().unsqueeze(1)
        scores = torch.topk(own_best.reshape(s["batch"], -1), s["beams"]).values.reshape(-1)
        return {"scores": scores, "tokens": None, "parents": None, "generated": None}

    return {"norm": norm, "linear": linear, "select": select}[case["kind"]]()

"""Operator cases: root-mean-square norm with a residual, routing to experts, and
the experts' products in 8 bits.

Transformer blocks of image networks add a branch to their stream, normalise the
sum, and send each token's row through an MLP.  With experts, a router's logits
choose a few of many MLPs for each token.  The cases below are those steps, with
their inputs and outputs in device memory:

  norm    the sum of two maps' rows and its root-mean-square norm
  norm8   the same, the norm in f16 and in 8 bits (e4m3 with a power-of-two scale
          for each 128 channels of a row), the latter read back as f16
  route   each token's experts and their weights from its logits, and the tokens
          in the order of their experts
  in8     the experts' first product of rows in 8 bits, with an activation (gated
          or not), in 8 bits, read back as f16
  out8    their second product, and each token's weighted sum of them
  mlp     norm8, route, in8 and out8 as a block runs them, with the residual

A pair is a token and one of its experts: token x top + slot, best expert first.
Rows between the two products are pairs in the order of their experts, a pair
without an expert (-1: none may be chosen) last.
"""

import functools
import importlib
import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-6
BLOCK = 128
TYPES = {"f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # One token's row on its way into a block: latency.
        dict(name="norm_1_768", kind="norm", rows=1, c=768, extra=0, into="f16", added="f16", outof="f16"),
        # A ragged map whose stream is kept in f32, its channels a part of each pixel's.
        dict(name="norm_10625_387", kind="norm", rows=10625, c=387, extra=5, into="f32", added="f16", outof="f16"),
        # The tokens of sixteen 1024 x 1024 images, a wide stream.
        dict(name="norm_65536_1024", kind="norm", rows=65536, c=1024, extra=0, into="f16", added="f16", outof="f16"),
        # A stage's tokens on their way into a router (f16) and its experts (8 bits).
        dict(name="norm8_16384_1536", kind="norm8", rows=16384, c=1536, extra=0, into="f16", added="f16", outof="f16"),
        # One token: latency.
        dict(name="route_1_64", kind="route", tokens=1, experts=64, top=8, score="softmax", bias=False, groups=1,
             kept=1, renorm=True, masked=False, into="f32"),
        # The tokens of a ragged map, some experts switched off.
        dict(name="route_10625_60", kind="route", tokens=10625, experts=60, top=4, score="softmax", bias=False,
             groups=1, kept=1, renorm=False, masked=True, into="f16"),
        # Many tokens and experts, balanced by a bias, in groups.
        dict(name="route_65536_256", kind="route", tokens=65536, experts=256, top=8, score="sigmoid", bias=True,
             groups=8, kept=4, renorm=True, masked=False, into="f32"),
        # One token through eight wide experts: their weights are read once.
        dict(name="in8_1_1024_2048", kind="in8", tokens=1, c=1024, hidden=2048, experts=64, top=8, gated=True,
             act="silu"),
        # The first layer of a transformer stage's MLP on a 64 x 64 map, two of sixteen experts.
        dict(name="in8_4096_384_1536", kind="in8", tokens=4096, c=384, hidden=1536, experts=16, top=2, gated=False,
             act="gelu"),
        # A second layer of odd widths, accumulated in f32.
        dict(name="out8_5000_1000_387", kind="out8", tokens=5000, c=387, hidden=1000, experts=20, top=3, outof="f32",
             add=True, extra=5),
        # A block over a few tokens, most experts with one or two of them.
        dict(name="mlp_32_1024_1024", kind="mlp", tokens=32, c=1024, hidden=1024, experts=64, top=4, gated=True,
             act="silu", score="softmax"),
        # A wide block over the tokens of four 1024 x 1024 images.
        dict(name="mlp_16384_1024_2048", kind="mlp", tokens=16384, c=1024, hidden=2048, experts=32, top=4, gated=True,
             act="silu", score="sigmoid"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "norm8", "route", "route", "in8", "in8", "out8", "out8", "mlp", "mlp"))
    if kind in ("norm", "norm8"):
        c = rng.choice((_log_int(rng, 1, 8192), 64 * rng.randint(1, 64)))
        return dict(kind=kind, rows=_log_int(rng, 1, min(1 << 17, 60 * 10**6 // c)), c=c, extra=rng.choice((0, 0, 8, 5)),
                    into=rng.choice(("f16", "f16", "f32")), added=rng.choice(("f16", "f32", "none")),
                    outof=rng.choice(("f16", "f16", "f32")) if kind == "norm" else "f16")
    if kind == "route":
        groups = rng.choice((1, 1, 1, 4, 8))
        experts = groups * rng.choice((_log_int(rng, 2, 64), 8, 16, 32))
        kept = rng.randint(1, groups)
        top = rng.randint(1, min(16, experts // groups * kept))
        return dict(kind=kind, tokens=_log_int(rng, 1, 65536), experts=experts, top=top,
                    score=rng.choice(("softmax", "sigmoid")), bias=rng.random() < 0.5, groups=groups, kept=kept,
                    renorm=rng.random() < 0.6, masked=rng.random() < 0.3, into=rng.choice(("f32", "f32", "f16")))
    while True:
        c = rng.choice((_log_int(rng, 16, 2048), 64 * rng.randint(1, 24)))
        hidden = rng.choice((_log_int(rng, 16, 4096), 128 * rng.randint(1, 24)))
        experts = rng.choice((_log_int(rng, 2, 64), 8, 16, 64))
        top = rng.randint(1, min(8, experts))
        tokens = _log_int(rng, 1, 16384)
        if 6.0 * tokens * top * c * hidden <= 8e11 and experts * c * hidden <= 1 << 26 and tokens * top * max(c, hidden) <= 1 << 27:
            break
    case = dict(kind=kind, tokens=tokens, c=c, hidden=hidden, experts=experts, top=top)
    if kind == "out8":
        return dict(case, outof=rng.choice(("f16", "f32")), add=rng.random() < 0.5, extra=rng.choice((0, 0, 8, 5)))
    case["gated"] = rng.random() < 0.5
    case["act"] = rng.choice(("silu", "gelu")) if case["gated"] else rng.choice(("gelu", "relu", "silu"))
    return case if kind == "in8" else dict(case, score=rng.choice(("softmax", "sigmoid")))


# ---- the plain forms -------------------------------------------------------------


def _blocks(k):
    return -(-k // BLOCK)


def _power(e):
    """2^e for whole e in -126 .. 127."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantize(x):
    """f32 rows [r, k] as e4m3 [r, blocks, 128] and exponents [r, blocks]."""
    r, k = x.shape
    x = torch.cat([x, x.new_zeros(r, _blocks(k) * BLOCK - k)], 1).reshape(r, -1, BLOCK)
    largest = x.abs().amax(2)
    m, e = torch.frexp(largest)  # m in 1/2 .. 1; 448 = 7/8 x 2^9
    e = torch.where(largest > 0, e.to(torch.int32) - 9 + (m > 0.875), 0)
    return (x * _power(-e)[:, :, None]).to(torch.float8_e4m3fn), e


def _values(q, e, k):
    """The f32 rows that _quantize's result stands for."""
    return (q.float() * _power(e)[:, :, None]).reshape(q.shape[0], -1)[:, :k]


def _in_eight(x):
    return _values(*_quantize(x), x.shape[1])


def _laid_out(q, e):
    """The bytes of rows in 8 bits: data [r, 128 blocks] and scales [r, a multiple of 4]."""
    r, blocks = e.shape
    scales = torch.full((r, 4 * -(-blocks // 4)), 127, dtype=torch.uint8, device=e.device)
    scales[:, :blocks] = (e + 127).to(torch.uint8)
    return q.view(torch.uint8).reshape(r, -1), scales


def _weights(w):
    """f32 weights [experts, c, n] as the f32 values of their 8-bit form."""
    experts, c, n = w.shape
    return _in_eight(w.transpose(1, 2).reshape(experts * n, c)).reshape(experts, n, c).transpose(1, 2).contiguous()


def _act(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return torch.relu(v)


def _hidden(v, act, gated):
    """f32 outputs of a first product, activated: of a gated one, act(first half) x second half."""
    half = v.shape[1] // 2
    return _act(v[:, :half], act) * v[:, half:] if gated else _act(v, act)


def _norm(x, added, gamma):
    """(the sum, its norm) in f32."""
    x = x.float() if added is None else x.float() + added.float()
    return x, x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * gamma


def _route(logits, top, score, bias, groups, kept, renorm, scale):
    """(experts [t, top], weights, offsets, order): scores in f64, whose last bits decide between two experts."""
    tokens, experts = logits.shape
    v = logits.double()
    v = torch.where(v.isnan(), -math.inf, v)
    open_ = v > -math.inf
    s = torch.sigmoid(v) if score == "sigmoid" else torch.softmax(torch.where(open_.any(1, keepdim=True), v, 0.0), 1)
    choice = torch.where(open_, s if bias is None else s + bias.double(), -math.inf)
    if groups > 1:
        best = torch.sort(choice.reshape(tokens, groups, -1), dim=2, descending=True).values[:, :, :1 if bias is None else 2]
        rank = torch.where(best[:, :, 0] > -math.inf, torch.where(best > -math.inf, best, 0.0).sum(2), -math.inf)
        order = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :kept]
        keep = torch.zeros_like(rank, dtype=torch.bool).scatter_(1, order, True)
        choice = torch.where(keep.repeat_interleave(experts // groups, 1), choice, -math.inf)
    choice, index = torch.sort(choice, dim=1, descending=True, stable=True)
    choice, index = choice[:, :top], index[:, :top]
    weight = torch.where(choice > -math.inf, s.gather(1, index), 0.0)
    if renorm:
        total = weight.sum(1, keepdim=True)
        weight = torch.where(total > 0, weight / total, 0.0)
    index = torch.where(choice > -math.inf, index, -1)
    return (index.int(), (scale * weight).float(), *_plan(index, experts))


def _plan(index, experts):
    """(offsets [experts + 1], order [pairs]) of experts [t, top]."""
    flat = torch.where(index < 0, experts, index).reshape(-1)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=index.device)
    offsets[1:] = torch.cumsum(torch.bincount(flat, minlength=experts + 1)[:experts], 0)
    return offsets, torch.sort(flat, stable=True).indices.int()


def _products(x, index, order, w, b):
    """f32 rows x, one a pair in the order of their experts, by their experts' weights."""
    expert = index.reshape(-1)[order.long()].long()
    pairs, experts = expert.numel(), w.shape[0]
    if pairs <= experts:
        return torch.bmm(x[:, None], w[expert])[:, 0] + b[expert]
    counts = torch.bincount(expert, minlength=experts)
    place = torch.arange(pairs, device=x.device) - (torch.cumsum(counts, 0) - counts)[expert]
    padded = x.new_zeros(experts, int(counts.max()), x.shape[1])
    padded[expert, place] = x
    return (torch.bmm(padded, w) + b[:, None])[expert, place]


def _combine(y, weight, order):
    """Each token's weighted sum of its pairs' f32 rows."""
    tokens, top = weight.shape
    by_pair = torch.empty_like(y)
    by_pair[order.long()] = y
    return (by_pair.reshape(tokens, top, -1) * weight[:, :, None]).sum(1)


# ---- what a program holds --------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _ien():
    return importlib.import_module("image-engine-native_amd.ien")


@functools.lru_cache(maxsize=None)
def _context():
    return _ien().Context(0)


def _features(g, rows, c):
    """What a stream holds: channels of their own mean and spread, a few far values."""
    x = torch.randn(rows, c, generator=g, device=DEVICE)
    x += 0.02 * x * x * x
    x *= 0.3 + 1.5 * torch.rand(c, generator=g, device=DEVICE)
    return x.add_(0.3 * torch.randn(c, generator=g, device=DEVICE))


def _held(x, extra, dtype):
    """Rows as `dtype` in a buffer with `extra` more columns, and the view of theirs."""
    buffer = torch.zeros(x.shape[0], x.shape[1] + extra, dtype=dtype, device=DEVICE)
    buffer[:, :x.shape[1]] = x
    return buffer[:, :x.shape[1]]


def _logits(g, tokens, experts):
    """A router's: some experts are liked better than others."""
    return torch.randn(tokens, experts, generator=g, device=DEVICE) + 0.5 * torch.randn(experts, generator=g, device=DEVICE)


def _layer(g, experts, c, n, gated=False):
    """Weights, as the f32 that a file holds, and biases."""
    w = torch.randn(experts, c, n, generator=g, device=DEVICE) / math.sqrt(c)
    b = 0.3 * torch.randn(experts, n, generator=g, device=DEVICE)
    if own:
        return dict(matrix=_ien().Experts8(_context(), w, b, gated=gated))
    return dict(w=_weights(w), b=b)


def _routes(g, case):
    """(experts, weights) of random tokens, and the plan."""
    logits = _logits(g, case["tokens"], case["experts"])
    value, index = torch.sort(logits, dim=1, descending=True, stable=True)
    index, weight = index[:, :case["top"]].int().contiguous(), torch.softmax(value[:, :case["top"]], 1).contiguous()
    if own:
        routes = _ien().Routes(case["tokens"], case["experts"], case["top"], index=index, weight=weight)
        _ien().plan_routes(_context(), routes)
        return dict(routes=routes)
    return dict(index=index, weight=weight, order=_plan(index, case["experts"])[1])


def prepare(case, seed):
    if own:
        _context()
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    kind, s = case["kind"], dict(case)
    if kind in ("norm", "norm8"):
        rows, c = case["rows"], case["c"]
        s["x"] = _held(_features(g, rows, c), case["extra"], TYPES[case["into"]])
        s["branch"] = None
        if case["added"] != "none":
            s["branch"] = _held(torch.randn(rows, c, generator=g, device=DEVICE), case["extra"], TYPES[case["added"]])
        s["gamma"] = 1 + 0.2 * torch.randn(c, generator=g, device=DEVICE)
        if own:
            s["sum"] = torch.empty(rows, c, dtype=TYPES[case["into"]], device=DEVICE)
            s["y"] = torch.empty(rows, c, dtype=TYPES[case["outof"]], device=DEVICE)
            if kind == "norm8":
                s["q"], s["back"] = _ien().Rows8(rows, c), torch.empty(rows, c, dtype=torch.float16, device=DEVICE)
    elif kind == "route":
        logits = _logits(g, case["tokens"], case["experts"])
        off = torch.rand(case["experts"], generator=g, device=DEVICE) < 0.2
        if case["masked"]:  # some experts for all tokens, all experts for some tokens
            logits[:, off] = -math.inf
            logits[::97] = -math.inf
        s["logits"] = logits.to(TYPES[case["into"]])
        s["offset"] = 0.1 * torch.randn(case["experts"], generator=g, device=DEVICE) if case["bias"] else None
        if own:
            s["routes"] = _ien().Routes(case["tokens"], case["experts"], case["top"])
    else:
        tokens, c, hidden, experts, top = (case[n] for n in ("tokens", "c", "hidden", "experts", "top"))
        if kind != "mlp":
            s.update(_routes(g, case))
        if kind != "out8":
            wide = hidden * (2 if case["gated"] else 1)
            s["first"] = _layer(g, experts, c, wide, case["gated"])
        if kind != "in8":
            s["second"] = _layer(g, experts, hidden, c)
        if kind == "mlp":
            s["x"] = _features(g, tokens, c).half()
            s["branch"] = torch.randn(tokens, c, generator=g, device=DEVICE).half()
            s["gamma"] = 1 + 0.2 * torch.randn(c, generator=g, device=DEVICE)
            s["logits"] = _logits(g, tokens, experts)
            s["offset"] = 0.1 * torch.randn(experts, generator=g, device=DEVICE)
            if own:
                s["q"] = _ien().Rows8(tokens, c)
                s["routes"] = _ien().Routes(tokens, experts, top)
        else:
            rows, k = (tokens, c) if kind == "in8" else (tokens * top, hidden)
            q, e = _quantize(_act(_features(g, rows, k), "silu"))
            if own:
                data, scales = _laid_out(q, e)
                s["q"] = _ien().Rows8(rows, k, data=data, scales=scales)
            else:
                s["q"], s["e"] = q, e
        dtype = TYPES[case.get("outof", "f16")]
        s["residual"] = None
        if kind == "out8" and case["add"]:
            s["residual"] = _held(torch.randn(tokens, c, generator=g, device=DEVICE), case["extra"], dtype)
        if own and kind != "out8":
            s["h"] = _ien().Rows8(tokens * top, hidden)
        if own and kind == "in8":
            s["y"] = torch.empty(tokens * top, hidden, dtype=dtype, device=DEVICE)
        elif own:
            s["parts"] = _ien().expert_parts(s["routes"], s["second"]["matrix"], torch.float32)
            s["y"] = _held(torch.zeros(tokens, c, device=DEVICE), case.get("extra", 0), dtype)
    return s


# ---- one pass --------------------------------------------------------------------


def _how(s):
    """A router's choices as keywords of the framework's call."""
    ien = _ien()
    return dict(score=ien.SCORE_SIGMOID if s["score"] == "sigmoid" else ien.SCORE_SOFTMAX, bias=s["offset"],
                groups=s.get("groups", 1), kept=s.get("kept", 1), group_top=1 if s["offset"] is None else 2,
                renormalise=s.get("renorm", True), scale=1.0 if s["score"] == "softmax" else 2.5)


def _run_own(s):
    ien, ctx, kind = _ien(), _context(), s["kind"]
    acts = dict(silu=ien.ACT_SILU, gelu=ien.ACT_GELU, relu=ien.ACT_RELU)
    if kind == "norm":
        ien.rms_norm(ctx, s["x"], s["gamma"], s["y"], add=s["branch"], total=s["sum"], eps=EPS)
        return s["sum"], s["y"]
    if kind == "norm8":
        ien.rms_norm(ctx, s["x"], s["gamma"], s["y"], s["q"], add=s["branch"], total=s["sum"], eps=EPS)
        ien.dequantize8(ctx, s["q"], s["back"])
        return s["sum"], s["y"], s["back"]
    if kind == "route":
        ien.route(ctx, s["logits"], s["routes"], **_how(s))
        r = s["routes"]
        return r.index, r.weight, r.offsets, r.order
    if kind == "in8":
        ien.experts_in8(ctx, s["q"], s["routes"], s["first"]["matrix"], s["h"], act=acts[s["act"]])
        ien.dequantize8(ctx, s["h"], s["y"])
    elif kind == "out8":
        ien.experts_out8(ctx, s["q"], s["routes"], s["second"]["matrix"], s["parts"], s["y"], add=s["residual"])
    else:
        ien.rms_norm(ctx, s["x"], s["gamma"], None, s["q"], add=s["branch"], eps=EPS)
        ien.route(ctx, s["logits"], s["routes"], **_how(s))
        ien.experts_in8(ctx, s["q"], s["routes"], s["first"]["matrix"], s["h"], act=acts[s["act"]])
        ien.experts_out8(ctx, s["h"], s["routes"], s["second"]["matrix"], s["parts"], s["y"], add=s["x"], branch=s["branch"])
    return s["y"]


def _run_plain(s):
    kind = s["kind"]
    if kind in ("norm", "norm8"):
        total, y = _norm(s["x"], s["branch"], s["gamma"])
        out = total.to(TYPES[s["into"]]), y.to(TYPES[s["outof"]])
        return out if kind == "norm" else (*out, _in_eight(y).half())
    if kind == "route":
        return _route(s["logits"], s["top"], s["score"], s["offset"], s["groups"], s["kept"], s["renorm"],
                      1.0 if s["score"] == "softmax" else 2.5)
    if kind == "in8":
        x = _values(s["q"], s["e"], s["c"])[s["order"].long() // s["top"]]
        v = _products(x, s["index"], s["order"], s["first"]["w"], s["first"]["b"])
        return _in_eight(_hidden(v, s["act"], s["gated"])).half()
    if kind == "out8":
        v = _products(_values(s["q"], s["e"], s["hidden"]), s["index"], s["order"], s["second"]["w"], s["second"]["b"])
        y = _combine(v, s["weight"], s["order"])
        return (y if s["residual"] is None else y + s["residual"].float()).to(TYPES[s["outof"]])
    total, n = _norm(s["x"], s["branch"], s["gamma"])
    index, weight, _, order = _route(s["logits"], s["top"], s["score"], s["offset"], 1, 1, True,
                                     1.0 if s["score"] == "softmax" else 2.5)
    x = _in_eight(n)[order.long() // s["top"]]
    v = _hidden(_products(x, index, order, s["first"]["w"], s["first"]["b"]), s["act"], s["gated"])
    v = _products(_in_eight(v), index, order, s["second"]["w"], s["second"]["b"])
    return (total + _combine(v, weight, order)).half()


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the work, and the results in 64 bits ----------------------------------------


def work(case):
    kind, size = case["kind"], {"f16": 2, "f32": 4, "none": 0}
    row8 = lambda k: k + _blocks(k)  # noqa: E731
    if kind in ("norm", "norm8"):
        n = case["rows"] * case["c"]
        moved = 2 * size[case["into"]] + size[case["added"]] + size[case["outof"]] + (2 if kind == "norm8" else 0)
        return dict(bytes=n * moved + 4 * case["c"], flops=5.0 * n)
    tokens, experts, top = case["tokens"], case["experts"], case["top"]
    routing = dict(bytes=tokens * (experts * size[case.get("into", "f32")] + 12 * top) + 4 * experts,
                   flops=tokens * experts * (4.0 + top))
    if kind == "route":
        return routing
    c, hidden, pairs = case["c"], case["hidden"], tokens * top
    used = experts * (1 - (1 - top / experts) ** tokens)  # experts with a token, on an average
    wide = hidden * (2 if case.get("gated") else 1)
    first = dict(bytes=used * wide * (row8(c) + 4), flops=2.0 * pairs * c * wide)
    second = dict(bytes=used * c * (row8(hidden) + 4), flops=2.0 * pairs * c * hidden)
    if kind == "in8":
        return dict(bytes=tokens * row8(c) + first["bytes"] + 2 * pairs * hidden, flops=first["flops"])
    if kind == "out8":
        written = tokens * c * size[case["outof"]] * (2 if case["add"] else 1)
        return dict(bytes=pairs * row8(hidden) + second["bytes"] + written, flops=second["flops"])
    return dict(bytes=6 * tokens * c + routing["bytes"] + first["bytes"] + second["bytes"],
                flops=routing["flops"] + first["flops"] + second["flops"])


def _exact_quantized(x):
    """f64 rows rounded to the 8-bit values, from the definition: the power of two of each block of 128 by
    comparing, the rounding by hand (a normal value has 4 significant bits, the smallest step is 2^-9)."""
    out = torch.zeros_like(x)
    for begin in range(0, x.shape[1], BLOCK):
        part = x[:, begin:begin + BLOCK]
        largest = part.abs().max(1).values
        e = torch.ceil(torch.log2(torch.where(largest > 0, largest, 1.0) / 448.0))
        e = torch.where(largest > 448.0 * torch.exp2(e), e + 1, e)
        e = torch.where(largest <= 448.0 * torch.exp2(e - 1), e - 1, e)
        unit = torch.exp2(torch.where(largest > 0, e, 0.0))[:, None]
        v = part / unit
        _, exponent = torch.frexp(v)
        step = torch.exp2((exponent - 4).clamp(min=-9).double())
        out[:, begin:begin + BLOCK] = torch.round(v / step) * step * unit
    return out


def _exact_act(y, act):
    if act == "silu":
        return y / (1 + torch.exp(-y))
    return y * torch.special.ndtr(y) if act == "gelu" else y.clamp(min=0)


def _exact_norm(x, added, gamma):
    v = x.double() if added is None else x.double() + added.double()
    return v, v / torch.sqrt(v.square().sum(1, keepdim=True) / v.shape[1] + EPS) * gamma.double()


def _exact_route(logits, top, score, bias, groups, kept, renorm, scale):
    """(experts, weights) in f64, a choice at a time: the best of what is left, the lowest index among equals."""
    tokens, experts = logits.shape
    at = torch.arange(tokens, device=logits.device)
    v = logits.double()
    closed = ~(v > -math.inf)
    if score == "sigmoid":
        s = 1 / (1 + torch.exp(-v))
    else:
        e = torch.where(closed, 0.0, torch.exp(v - v.max(1, keepdim=True).values))
        s = e / e.sum(1, keepdim=True)
    left = s.clone() if bias is None else s + bias.double()
    left[closed] = -math.inf
    if groups > 1:
        per = experts // groups
        rank = torch.zeros(tokens, groups, dtype=torch.float64, device=logits.device)
        for j in range(groups):
            part = left[:, j * per:(j + 1) * per].clone()
            for i in range(1 if bias is None else min(2, per)):
                best = part.max(1).values
                rank[:, j] += torch.where(best > -math.inf, best, -math.inf if i == 0 else 0.0)
                part[at, part.argmax(1)] = -math.inf
        out = torch.ones(tokens, groups, dtype=torch.bool, device=logits.device)
        for _ in range(kept):
            best = _first_best(rank)
            out[at, best] = False
            rank[at, best] = -math.inf
        for j in range(groups):
            left[:, j * per:(j + 1) * per][out[:, j]] = -math.inf
    index, weight = [], []
    for _ in range(top):
        best = _first_best(left)
        some = left[at, best] > -math.inf
        index.append(torch.where(some, best, -1))
        weight.append(torch.where(some, s[at, best], 0.0))
        left[at, best] = -math.inf
    index, weight = torch.stack(index, 1), torch.stack(weight, 1)
    if renorm:
        weight = weight / weight.sum(1, keepdim=True).clamp(min=1e-300)
    return index, scale * weight


def _first_best(v):
    best = v.max(1, keepdim=True).values
    n = torch.arange(v.shape[1], device=v.device)
    return torch.where(v == best, n, v.shape[1]).min(1).values


def exact(case, seed):
    kind = case["kind"]
    if kind == "in8":
        # A value that 32 bits put on the other side of a border between two 8-bit values is off by a sixteenth of
        # itself, on either side; a map of millions holds a few.
        return None
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    if kind in ("norm", "norm8"):
        x = _features(g, case["rows"], case["c"]).to(TYPES[case["into"]])
        branch = None
        if case["added"] != "none":
            branch = torch.randn(case["rows"], case["c"], generator=g, device=DEVICE).to(TYPES[case["added"]])
        total, y = _exact_norm(x, branch, 1 + 0.2 * torch.randn(case["c"], generator=g, device=DEVICE))
        return (total, y) if kind == "norm" else (total, y, None)
    scale = 1.0 if case.get("score") == "softmax" else 2.5
    if kind == "route":
        logits = _logits(g, case["tokens"], case["experts"])
        off = torch.rand(case["experts"], generator=g, device=DEVICE) < 0.2
        if case["masked"]:
            logits[:, off] = -math.inf
            logits[::97] = -math.inf
        bias = 0.1 * torch.randn(case["experts"], generator=g, device=DEVICE) if case["bias"] else None
        _, weight = _exact_route(logits.to(TYPES[case["into"]]), case["top"], case["score"], bias, case["groups"],
                                 case["kept"], case["renorm"], scale)
        return None, weight, None, None
    tokens, c, hidden, experts, top = (case[n] for n in ("tokens", "c", "hidden", "experts", "top"))

    def layer(c, n):
        w = torch.randn(experts, c, n, generator=g, device=DEVICE) / math.sqrt(c)
        return w, 0.3 * torch.randn(experts, n, generator=g, device=DEVICE)

    def product(x, i, w, b):
        return x @ _exact_quantized(w[i].double().t().contiguous()).t() + b[i].double()

    y = torch.zeros(tokens, c, dtype=torch.float64, device=DEVICE)
    if kind == "out8":
        logits = _logits(g, tokens, experts)
        value, index = torch.sort(logits, dim=1, descending=True, stable=True)
        index, weight = index[:, :top], torch.softmax(value[:, :top], 1).double()
        w, b = layer(hidden, c)
        x = _exact_quantized(_act(_features(g, tokens * top, hidden), "silu").double())
        begin = 0
        for i in range(experts):
            t, slot = torch.nonzero(index == i, as_tuple=True)  # (in the order of the tokens)
            y[t] += weight[t, slot, None] * product(x[begin:begin + t.numel()], i, w, b)
            begin += t.numel()
        if case["add"]:
            y += torch.randn(tokens, c, generator=g, device=DEVICE).to(TYPES[case["outof"]]).double()
        return y
    first, second = layer(c, hidden * (2 if case["gated"] else 1)), layer(hidden, c)
    x, branch = _features(g, tokens, c).half(), torch.randn(tokens, c, generator=g, device=DEVICE).half()
    total, n = _exact_norm(x, branch, 1 + 0.2 * torch.randn(c, generator=g, device=DEVICE))
    n, logits = _exact_quantized(n), _logits(g, tokens, experts)
    bias = 0.1 * torch.randn(experts, generator=g, device=DEVICE)
    index, weight = _exact_route(logits, top, case["score"], bias, 1, 1, True, scale)
    for i in range(experts):
        t, slot = torch.nonzero(index == i, as_tuple=True)
        v = product(n[t], i, *first)
        v = _exact_act(v[:, :hidden], case["act"]) * v[:, hidden:] if case["gated"] else _exact_act(v, case["act"])
        y[t] += weight[t, slot, None] * product(_exact_quantized(v), i, *second)
    return total + y

"""Operators of the library as cases that can be timed and compared: weights in 8-bit floating point with a scale for each
block of 128 x 128, as a dense projection and as a mixture's experts, and the router in front of those.

  product  y = x W^T.  W holds OCP E4M3 codes and an f32 scale for every 128 rows x 128 columns; every 128 columns of an
           activation row are quantized to E4M3 within the call, under the smallest power of two that brings their largest
           magnitude to 448 or less (not below 2^-100).  f32 in, f32 out.
  experts  the same over groups of rows: pair p of group g (off[g] <= p < off[g + 1]) is row gather[p] of x times matrix g
           of a stack.
  route    every token's k best experts: scores softmax(l) or sigmoid(l) in 64 bits; with a bias, score + bias decides the
           choice; with groups of experts, the best groups (by the sum of their one or two best) are chosen first; the
           weights are the chosen experts' scores without the bias, divided by their sum where `norm` says so, times a
           factor.  Equal values go to the lowest index; an expert whose logit is -inf is not chosen, a slot without an
           expert holds id -1 and weight 0.

A case is a dict of plain values; `prepare` makes what a program holds before the call, `run` is one pass.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
BLOCK = 128


def listed():
    return [
        # one token of Llama-3-8B through the attention's output projection: the smallest product, latency counts
        {"name": "product_decode", "family": "product", "batch": 1, "rows": 4096, "cols": 4096},
        # one token through its gate (or up) projection: the weights' bytes count
        {"name": "product_decode_wide", "family": "product", "batch": 1, "rows": 14336, "cols": 4096},
        # eight sequences decoding together, the down projection
        {"name": "product_batch_8", "family": "product", "batch": 8, "rows": 4096, "cols": 14336},
        # an odd number of sequences; neither rows nor columns are whole blocks (gpt-oss-20b's width, 22 blocks and a half)
        {"name": "product_batch_61_ragged", "family": "product", "batch": 61, "rows": 2880, "cols": 2880},
        # a 512-token prompt chunk, gate or up
        {"name": "product_prefill", "family": "product", "batch": 512, "rows": 14336, "cols": 4096},
        # a long prompt's down projection: the largest
        {"name": "product_prefill_long", "family": "product", "batch": 4096, "rows": 4096, "cols": 14336},
        # one token through a projection of 8 of 128 experts (Qwen3-30B-A3B's shapes)
        {"name": "experts_decode", "family": "experts", "tokens": 1, "experts": 128, "top_k": 8, "rows": 768, "cols": 2048},
        # a 512-token chunk through the same: every expert is read, for about 32 pairs each
        {"name": "experts_prefill", "family": "experts", "tokens": 512, "experts": 128, "top_k": 8, "rows": 768, "cols": 2048},
        # a long prompt through 32 experts of gpt-oss-20b's width, top-4: about 256 pairs each
        {"name": "experts_prefill_long", "family": "experts", "tokens": 2048, "experts": 32, "top_k": 4, "rows": 2880, "cols": 2880},
        # the router of one token: 128 experts, softmax, the top eight's weights renormalised
        {"name": "route_decode", "family": "route", "tokens": 1, "experts": 128, "top_k": 8, "score": "softmax", "bias": False,
         "groups": 1, "top_groups": 1, "group_best": 1, "norm": True, "scale": 1.0},
        # a 512-token chunk: 256 experts in 8 groups of which 4 are used, sigmoid scores and a bias for balance
        {"name": "route_grouped", "family": "route", "tokens": 512, "experts": 256, "top_k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_best": 2, "norm": True, "scale": 2.5},
        # a batch of long prompts, the same router
        {"name": "route_grouped_long", "family": "route", "tokens": 16384, "experts": 256, "top_k": 8, "score": "sigmoid", "bias": True,
         "groups": 8, "top_groups": 4, "group_best": 2, "norm": True, "scale": 2.5},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    family = rng.choice(("product", "product", "experts", "route"))
    if family == "product":
        def width():
            # whole blocks as in most models, halves of blocks, or anything
            kind, n = rng.random(), _log_int(rng, 96, 14336)
            return max(BLOCK, n // BLOCK * BLOCK) if kind < 0.5 else max(64, n // 64 * 64) if kind < 0.75 else n
        rows, cols = width(), width()
        return {"family": family, "batch": _log_int(rng, 1, min(4096, 4096 * 4096 * 14336 // (rows * cols))), "rows": rows, "cols": cols}
    if family == "experts":
        experts, k = rng.choice((8, 16, 32, 60, 64, 128)), rng.choice((1, 2, 4, 6, 8))
        rows, cols = _log_int(rng, 100, 2880), 32 * _log_int(rng, 4, 90)
        tokens = _log_int(rng, 1, min(2048, 2048 * 4 * 2880 * 2880 // (k * rows * cols)))
        if experts * rows * cols > 32 * 2880 * 2880:
            rows = 32 * 2880 * 2880 // (experts * cols)
        return {"family": family, "tokens": tokens, "experts": experts, "top_k": k, "rows": rows, "cols": cols}
    grouped = rng.random() < 0.5
    groups = rng.choice((2, 4, 8)) if grouped else 1
    experts = groups * _log_int(rng, 8, 512 // groups)
    top_groups = rng.randint(1, groups)
    return {"family": family, "tokens": _log_int(rng, 1, min(16384, 16384 * 256 // experts)), "experts": experts,
            "top_k": rng.randint(1, min(10, top_groups * (experts // groups))), "score": rng.choice(("softmax", "sigmoid")),
            "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups, "group_best": rng.choice((1, 2)) if grouped else 1,
            "norm": rng.random() < 0.7, "scale": rng.choice((1.0, 2.5))}


# ---- inputs ----

def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _expand(scales, rows, cols):
    """[..., row blocks, column blocks] as [..., rows, cols]."""
    return scales.repeat_interleave(BLOCK, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :cols]


def _weights(gen, matrices, rows, cols):
    """Matrices of N(0, 0.02) weights whose spread differs from block to block, quantized as checkpoints of this kind are: an
    f32 scale that takes a block's largest magnitude to 448."""
    w = torch.empty((matrices, rows, cols), dtype=torch.float8_e4m3fn, device=DEVICE)
    scales = torch.empty((matrices, _blocks(rows), _blocks(cols)), dtype=torch.float32, device=DEVICE)
    step = max(1, (1 << 27) // (rows * cols))  # (matrices at a time)
    for m in range(0, matrices, step):
        n = min(step, matrices - m)
        spread = torch.rand((n, _blocks(rows), _blocks(cols)), generator=gen, device=DEVICE) * 0.03 + 0.005
        v = torch.randn((n, rows, cols), generator=gen, device=DEVICE) * _expand(spread, rows, cols)
        s = spread * (4.2 / 448)
        scales[m:m + n] = s
        w[m:m + n] = (v / _expand(s, rows, cols)).clamp_(-448, 448).to(torch.float8_e4m3fn)
    return w, scales


def _activations(gen, rows, cols):
    """Normalised hidden states: N(0, 1), a few channels eight times as large."""
    x = torch.randn((rows, cols), generator=gen, device=DEVICE)
    x[:, torch.randint(0, cols, (max(1, cols // 512),), generator=gen, device=DEVICE)] *= 8.0
    return x


def prepare(case, seed):
    gen = torch.Generator(DEVICE)
    gen.manual_seed(seed)
    family = case["family"]
    s = {"family": family, "case": case}
    if family == "route":
        s["logits"] = torch.randn((case["tokens"], case["experts"]), generator=gen, device=DEVICE) * 1.5
        s["bias"] = torch.randn(case["experts"], generator=gen, device=DEVICE) * 0.1 if case["bias"] else None
        return s
    rows, cols = case["rows"], case["cols"]
    if family == "product":
        s["w"], s["scales"] = _weights(gen, 1, rows, cols)
        s["x"] = _activations(gen, case["batch"], cols)
    else:
        e, t, k = case["experts"], case["tokens"], case["top_k"]
        s["w"], s["scales"] = _weights(gen, e, rows, cols)
        s["x"] = _activations(gen, t, cols)
        # what a router and a sort of its choices leave: the pairs of every expert, tokens ascending
        ids = torch.randn((t, e), generator=gen, device=DEVICE).topk(k, dim=1).indices.flatten()
        s["gather"] = (ids.argsort(stable=True) // k).to(torch.int32)
        counts = torch.bincount(ids, minlength=e)
        s["off"] = torch.cat((counts.new_zeros(1), counts.cumsum(0))).to(torch.int32)
        s["most"] = int(counts.max())
    if own:  # the resident copy that a program makes of its weights when it loads them
        import frink_amd as fa
        s["resident"] = fa.Weights.from_device_fp8(s["w"], s["scales"], s["w"].shape[0] * rows, cols, matrices=s["w"].shape[0])
    return s


# ---- the plain forms ----

def _quantized(x):
    """x's values after their quantization, in f32."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x, (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    mantissa, exponent = torch.frexp(v.abs().amax(-1, keepdim=True))  # amax = mantissa 2^exponent; 448 = 0.875 x 2^9
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(min=-100)
    up, down = ((127 - e) << 23).view(torch.float32), ((127 + e) << 23).view(torch.float32)
    return ((v * up).to(torch.float8_e4m3fn).to(torch.float32) * down).view(rows, -1)[:, :cols]


def _scores(logits, score):
    l = logits.double()
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-l))
    p = torch.exp(l - l.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _first(values, n):
    """The indices of the n largest along the last axis, equal ones in ascending order."""
    return values.sort(dim=-1, descending=True, stable=True).indices[..., :n]


def _route(logits, bias, c):
    t, e, g = c["tokens"], c["experts"], c["groups"]
    p = _scores(logits, c["score"])
    choice = p if bias is None else p + bias.double()
    choice = torch.where(logits > -math.inf, choice, -math.inf)
    if g > 1:
        best = choice.view(t, g, e // g).sort(dim=-1, descending=True).values[..., :c["group_best"]]
        some = best[..., :1] > -math.inf
        value = torch.where(some, torch.where(best > -math.inf, best, 0.0).sum(-1, keepdim=True), -math.inf)[..., 0]
        used = torch.zeros_like(value, dtype=torch.bool).scatter_(1, _first(value, c["top_groups"]), True)
        choice = torch.where(used.repeat_interleave(e // g, 1), choice, -math.inf)
    ids = _first(choice, c["top_k"])
    there = choice.gather(1, ids) > -math.inf
    w = torch.where(there, p.gather(1, ids), 0.0)
    if c["norm"]:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return torch.where(there, ids, -1).to(torch.int32), (w * c["scale"]).to(torch.float32)


def _experts(s):
    w, x, off, gather = s["w"], s["x"], s["off"].long(), s["gather"].long()
    n, rows, cols = w.shape
    pairs = gather.numel()
    a = _quantized(x)[gather]
    group = torch.searchsorted(off[1:], torch.arange(pairs, device=DEVICE), right=True)
    if pairs <= n:  # every pair with its own copy of its matrix
        m = w.view(torch.uint8)[group].view(torch.float8_e4m3fn).to(torch.float32) * _expand(s["scales"][group], rows, cols)
        return torch.bmm(m, a[:, :, None])[:, :, 0]
    # all groups as long as the longest
    at = group * s["most"] + torch.arange(pairs, device=DEVICE) - off[group]
    padded = torch.zeros((n * s["most"], cols), device=DEVICE)
    padded[at] = a
    m = w.to(torch.float32) * _expand(s["scales"], rows, cols)
    y = torch.bmm(m, padded.view(n, s["most"], cols).transpose(1, 2).contiguous())
    return y.transpose(1, 2).reshape(-1, rows)[at]


def run(s):
    c, family = s["case"], s["family"]
    if own:
        import frink_amd as fa
        if family == "product":
            return s["resident"].gemm(s["x"])
        if family == "experts":
            return fa.gemm_grouped(s["resident"], c["experts"], s["off"], s["x"], gather=s["gather"])
        return fa.route(s["logits"], c["top_k"], score=c["score"], bias=s["bias"], groups=c["groups"], top_groups=c["top_groups"],
                        group_best=c["group_best"], norm=c["norm"], scale=c["scale"])
    if family == "product":
        m = s["w"][0].to(torch.float32) * _expand(s["scales"][0], c["rows"], c["cols"])
        return _quantized(s["x"]) @ m.T
    if family == "experts":
        return _experts(s)
    return _route(s["logits"], s["bias"], c)


# ---- what a pass cannot do without ----

def work(case):
    if case["family"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        return {"bytes": 4 * (t * (e + 2 * k) + (e if case["bias"] else 0)), "flops": 8 * t * e}
    rows, cols = case["rows"], case["cols"]
    matrix = rows * cols + 4 * _blocks(rows) * _blocks(cols)
    if case["family"] == "product":
        return {"bytes": matrix + 4 * case["batch"] * (rows + cols), "flops": 2 * case["batch"] * rows * cols}
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    visited = e * (1.0 - (1.0 - k / e) ** t)  # the experts that independent choices of t tokens are expected to reach
    return {"bytes": visited * matrix + 4 * (t * cols + t * k * (rows + 1) + e + 1), "flops": 2 * t * k * rows * cols}


# ---- the definition in 64 bits ----

def _quantized64(x):
    x = x.double()
    out = torch.empty_like(x)
    for k in range(0, x.shape[1], BLOCK):
        v = x[:, k:k + BLOCK]
        top = v.abs().max(1, keepdim=True).values
        e = torch.ceil(torch.log2(torch.where(top > 0, top, 1.0) / 448.0))
        for d in (-1.0, 1.0):  # (the logarithm's own rounding)
            e = torch.where((top <= 448.0 * 2.0 ** (e - 1)) if d < 0 else (top > 448.0 * 2.0 ** e), e + d, e)
        e = e.clamp(min=-100.0)
        z = v * 2.0 ** -e
        # E4M3: three bits behind the leading one, its exponent at least -6; halves to the even neighbour
        step = 2.0 ** (torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3.0)
        out[:, k:k + BLOCK] = torch.round(z / step) * step * 2.0 ** e
    return out


def _exact_route(logits, bias, c):
    l = logits.double()
    if c["score"] == "sigmoid":
        p = torch.where(l >= 0, 1.0 / (1.0 + torch.exp(-l.abs())), torch.exp(-l.abs()) / (1.0 + torch.exp(-l.abs())))
    else:
        p = torch.exp(l - torch.logsumexp(l, 1, keepdim=True))
    value = p + (0.0 if bias is None else bias.double())
    value[logits == -math.inf] = -math.inf
    size = c["experts"] // c["groups"]
    if c["groups"] > 1:
        score = torch.stack([value[:, g * size:(g + 1) * size].topk(min(size, c["group_best"]), dim=1).values.clamp(min=-1e300).sum(1)
                             for g in range(c["groups"])], 1)
        for _ in range(c["groups"] - c["top_groups"]):  # the worst group goes, of equal ones the last
            worst = c["groups"] - 1 - score.flip(1).argmin(1)
            score.scatter_(1, worst[:, None], math.inf)
            mine = torch.arange(c["experts"], device=DEVICE)[None] // size == worst[:, None]
            value[mine] = -math.inf
    ids, weights = [], []
    for _ in range(c["top_k"]):
        top, at = value.max(1)
        first = (value == top[:, None]).double().argmax(1)
        gone = top == -math.inf
        ids.append(torch.where(gone, -1, first))
        weights.append(torch.where(gone, 0.0, p.gather(1, first[:, None])[:, 0]))
        value.scatter_(1, first[:, None], -math.inf)
    w = torch.stack(weights, 1)
    if c["norm"]:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
    return torch.stack(ids, 1).to(torch.int32), w * c["scale"]


def exact(case, seed):
    s = prepare(case, seed)
    if case["family"] == "route":
        return _exact_route(s["logits"], s["bias"], case)
    rows, cols = case["rows"], case["cols"]
    a = _quantized64(s["x"])

    def matrix(g):
        m = s["w"][g].double()
        for r in range(_blocks(rows)):
            for k in range(_blocks(cols)):
                m[r * BLOCK:(r + 1) * BLOCK, k * BLOCK:(k + 1) * BLOCK] *= s["scales"][g, r, k].double()
        return m
    if case["family"] == "product":
        return a @ matrix(0).T
    off, gather = s["off"].tolist(), s["gather"].long()
    y = torch.empty((gather.numel(), rows), dtype=torch.float64, device=DEVICE)
    for g in range(case["experts"]):
        if off[g + 1] > off[g]:
            y[off[g]:off[g + 1]] = a[gather[off[g]:off[g + 1]]] @ matrix(g).T
    return y

"""What is timed of the operators of low-bit serving: keys and values held in 4 bits, and
products of rows and weights in 8 bits.

A case is one call of one operator.  `kind`:

"attend"   paged attention over a cache in 4 bits.  `lanes` requests bring one token each, their
           contexts spread from `ctx_lo` to `ctx_hi` tokens; `portions` is a text "start+tokens,..."
           of further requests that bring a portion of a prompt behind `start` cached tokens.
"store"    the keys and values of a step's tokens go into such a cache and are read back as the
           values it holds (`lanes` and `portions` as above).
"linear"   rows [M, K] times a weight [N, K] in 8 bits, rows quantised within the call.
"gate_up"  add, RMSNorm, 8-bit rows, the product with a stacked gate/up weight [2 N, K] and
           silu(gate) * up: what stands in front of a feed-forward's second product.

The 4-bit form: a group is up to 64 neighbouring elements of a head of one token; its step is a
fifteenth of the way from its smallest element (or zero, if that is less) to its largest (or
zero) in float16, its zero the whole number of steps nearest to that way's share below zero, and
an element is held as the nearest of step * (0 - zero .. 15 - zero).  The 8-bit form: a
row's scale is its largest magnitude / 127, an element the nearest whole number of scales.
"""

from __future__ import annotations

import math

import torch

own = False

GROUP = 64
DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases


def _attend(name, heads, kv_heads, dim, page, dtype="bf16", lanes=0, ctx_lo=0, ctx_hi=0,
            portions="", window=0):
    case = dict(kind="attend", heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                lanes=lanes, ctx_lo=ctx_lo, ctx_hi=ctx_hi, portions=portions, window=window)
    return case if name is None else dict(name=name, **case)


def _store(name, kv_heads, dim, page, dtype="bf16", lanes=0, ctx_lo=0, ctx_hi=0, portions=""):
    case = dict(kind="store", kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, lanes=lanes,
                ctx_lo=ctx_lo, ctx_hi=ctx_hi, portions=portions)
    return case if name is None else dict(name=name, **case)


def _product(name, kind, rows, columns, inner, dtype="bf16"):
    case = dict(kind=kind, M=rows, N=columns, K=inner, dtype=dtype)
    return case if name is None else dict(name=name, **case)


def listed():
    return [
        # one user waiting for the next token of the 0.6B preset: latency
        _attend("attend 1 of 541", 16, 8, 128, 16, lanes=1, ctx_lo=541, ctx_hi=541),
        # the 8B preset's server batch, contexts of all lengths
        _attend("attend 64 to 4096", 32, 8, 128, 16, lanes=64, ctx_lo=128, ctx_hi=4096),
        # a few long documents at the 32B preset, what a 4-bit cache makes room for
        _attend("attend 12 of 40000", 64, 8, 128, 64, lanes=12, ctx_lo=30011, ctx_hi=40960),
        # float32 activations, heads of 64, a window
        _attend("attend 24 fp32", 16, 4, 64, 16, "fp32", lanes=24, ctx_lo=100, ctx_hi=2047,
                window=1024),
        # a server's mixed step: odd portions behind odd lengths beside single tokens
        _attend("attend mixed", 16, 8, 128, 16, lanes=37, ctx_lo=1, ctx_hi=2000,
                portions="0+501,777+37,2048+1290"),
        # half of a long prompt of the 8B preset behind the other half
        _attend("attend prompt 4096", 32, 8, 128, 16, portions="4096+4096"),
        # the new tokens of a decode step
        _store("store 64", 8, 128, 16, lanes=64, ctx_lo=128, ctx_hi=4096),
        # a prompt's step at the largest token budget of the engine's defaults, two halves
        _store("store prompts", 8, 128, 16, portions="0+8191,333+8193"),
        # the 8B preset's output projection for one token: latency and the weight's bytes
        _product("linear 1 row", "linear", 1, 4096, 4096),
        # the 32B preset's q/k/v projection of a long prompt's portion: the matrix cores
        _product("linear 8192 rows", "linear", 8192, 10240, 5120),
        # the 8B preset's feed-forward in a decode step of 16 requests
        _product("gate_up 16 rows", "gate_up", 16, 12288, 4096),
        # the smaller of the hybrid sizes that bench.py compares, a portion of an odd length
        _product("gate_up 777 rows", "gate_up", 777, 4096, 1024),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    heads, kv_heads, dim = rng.choice([(16, 8, 128), (32, 8, 128), (64, 8, 128), (16, 4, 64),
                                       (8, 2, 256), (12, 3, 96), (6, 6, 80), (20, 1, 128)])
    page = rng.choice([16, 16, 32, 64, 256])
    kind = rng.choice(["decode", "decode", "long decode", "decode fp32", "mixed", "prompt",
                       "store", "store", "linear", "linear", "gate_up", "gate_up"])
    if kind in ("decode", "long decode", "decode fp32"):
        hi = 30000 if kind == "long decode" else 3500
        a, b = sorted((log_int(hi // 100, hi), log_int(hi // 100, hi)))
        lanes = log_int(1, 8) if kind == "long decode" else log_int(1, 64)
        return _attend(None, heads, kv_heads, dim, page, "fp32" if kind == "decode fp32" else "bf16",
                       lanes=lanes, ctx_lo=a, ctx_hi=b, window=rng.choice([0, 0, 0, 777]))
    if kind == "mixed":
        return _attend(None, heads, kv_heads, dim, page, lanes=log_int(1, 40), ctx_lo=1,
                       ctx_hi=log_int(2, 2000),
                       portions=f"{log_int(1, 1500) - 1}+{log_int(2, 900)},0+{log_int(1, 700)}",
                       window=rng.choice([0, 0, 300]))
    if kind == "prompt":
        return _attend(None, heads, kv_heads, dim, page, rng.choice(["bf16", "bf16", "fp32"]),
                       portions=f"{rng.choice([0, 0, 1, 800])}+{log_int(17, 1900)}")
    if kind == "store":
        return _store(None, kv_heads, dim, page, rng.choice(["bf16", "bf16", "fp32"]),
                      lanes=log_int(1, 200), ctx_lo=1, ctx_hi=log_int(1, 4000),
                      portions=rng.choice(["", f"{log_int(1, 999) - 1}+{log_int(1, 6000)}"]))
    if kind == "linear":
        return _product(None, "linear", log_int(1, 3000), log_int(33, 11000), log_int(64, 6000),
                        rng.choice(["bf16", "bf16", "fp32"]))
    return _product(None, "gate_up", log_int(1, 2000), 8 * log_int(16, 1500), 8 * log_int(16, 600))


def _requests(case):
    """(start, tokens) of every request of a step: the lanes, then the portions."""
    n, lo, hi = case["lanes"], case["ctx_lo"], case["ctx_hi"]
    # spread evenly and out of order, as requests come
    ctx = [lo + (hi - lo) * ((i * 37) % n) // max(n - 1, 1) for i in range(n)]
    out = [(c - 1, 1) for c in ctx]
    for part in filter(None, case["portions"].split(",")):
        start, tokens = part.split("+")
        out.append((int(start), int(tokens)))
    return out


def _groups(dim):
    return -(-dim // GROUP)


def work(case):
    size = 2 if case.get("dtype") == "bf16" else 4
    if case["kind"] in ("linear", "gate_up"):
        M, N, K = case["M"], case["N"], case["K"]
        two = 2 if case["kind"] == "gate_up" else 1
        # rows in (gate_up: the float32 stream in and out and what is added), weight and its
        # scales, the norm's weight, results
        rows = M * K * (4 + 4 + size) + 4 * K if two == 2 else M * K * size
        return {"bytes": rows + two * N * (K + 4) + M * N * size, "flops": 2.0 * two * M * N * K}
    held = case["dim"] / 2 + 4 * _groups(case["dim"])       # bytes of a key or value
    requests = _requests(case)
    tokens = sum(n for _, n in requests)
    if case["kind"] == "store":
        values = 2 * tokens * case["kv_heads"]
        return {"bytes": values * (2 * case["dim"] * size + 2 * held), "flops": 4.0 * values * case["dim"]}
    window = case["window"] or 1 << 40
    keys = sum(min(s + n, window + n - 1) for s, n in requests)
    pairs = sum(min(s + i + 1, window) for s, n in requests for i in range(n))
    return {"bytes": 2 * keys * case["kv_heads"] * held + 2 * tokens * case["heads"] * case["dim"] * size,
            "flops": 4.0 * pairs * case["heads"] * case["dim"]}


# ------------------------------------------------------------------ inputs


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEVICE)


def _heads_of(g, tokens, case):
    """Keys and values of `tokens` tokens, [tokens, kv_heads, dim]: keys have channels of larger
    magnitude, as keys behind a rotation do; values are smaller and even."""
    kv, dim = case["kv_heads"], case["dim"]
    loud = 1 + 4 * (torch.arange(dim, device=DEVICE) % 29 == 3)
    k = (_randn(g, tokens, kv, dim) * loud).to(TYPES[case["dtype"]])
    v = (0.5 * _randn(g, tokens, kv, dim)).to(TYPES[case["dtype"]])
    return k, v


def _step_inputs(case, seed):
    """(requests, block table, per request its keys and values in the cache's order, queries)."""
    g = _generator(seed)
    requests, P = _requests(case), case["page"]
    pages = [-(-(s + n) // P) for s, n in requests]
    order = torch.randperm(sum(pages), generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((len(requests), max(pages)), -1, dtype=torch.int32, device=DEVICE)
    first = 0
    for e, n in enumerate(pages):
        table[e, :n] = order[first:first + n]
        first += n
    tokens = sum(n for _, n in requests)
    held = [_heads_of(g, (s + n) if case["kind"] == "attend" else n, case) for s, n in requests]
    q = None
    if case["kind"] == "attend":
        q = _randn(g, tokens, case["heads"], case["dim"]).to(TYPES[case["dtype"]])
    return requests, table, held, q


def _product_inputs(case, seed):
    g = _generator(seed)
    M, N, K, t = case["M"], case["N"], case["K"], TYPES[case["dtype"]]
    two = 2 if case["kind"] == "gate_up" else 1
    # rows as they come out of a norm or an activation: some columns are louder than others
    loud = 1 + 3 * (torch.arange(K, device=DEVICE) % 61 == 7)
    w = (0.02 * _randn(g, two * N, K)).to(t)
    if two == 1:
        return dict(x=(_randn(g, M, K) * loud).to(t), w=w)
    return dict(resid=2 * _randn(g, M, K) * loud, delta=(0.3 * _randn(g, M, K)).to(t),
                norm=1 + 0.2 * _randn(g, K), w=w)


EPS = 1e-6


# ------------------------------------------------------------------ plain forms


def _quantize4(x):
    """[..., dim] -> codes [..., dim] (uint8), step (float16) and zero [..., groups]."""
    dim, n = x.shape[-1], _groups(x.shape[-1])
    # (zeros fill the last group up: zero is among what every group spans)
    wide = torch.nn.functional.pad(x.float(), (0, n * GROUP - dim)).unflatten(-1, (n, GROUP))
    least, most = wide.amin(-1).clamp(max=0.0), wide.amax(-1).clamp(min=0.0)
    step = ((most - least) / torch.full((), 15.0, device=x.device)).clamp(max=65504.0).half()
    # the border between two codes is decided in 64 bits
    by = step.double().where(step > 0, torch.ones((), dtype=torch.double, device=x.device))
    zero = (-least.double() / by).round().clamp(max=15).where(step > 0, by - by)
    c = (wide.double() / by[..., None]).round() + zero[..., None]
    c = c.clamp(0, 15).where(step[..., None] > 0, c - c)
    return c.flatten(-2)[..., :dim].to(torch.uint8), step, zero.to(torch.uint8)


def _values4(codes, step, zero):
    dim = codes.shape[-1]
    s = step.float().repeat_interleave(GROUP, -1)[..., :dim]
    return s * (codes.float() - zero.float().repeat_interleave(GROUP, -1)[..., :dim])


def _quantize8(x):
    """[rows, K] -> whole numbers (float64) and float32 scales."""
    scale = x.float().abs().amax(-1) / torch.full((), 127.0, device=x.device)
    code = x.double() / scale.double().clamp(min=1e-300)[:, None]
    return code.round(), scale


def _rms(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _plain_attend(s):
    case, out = s["case"], []
    kv, dim, P = case["kv_heads"], case["dim"], case["page"]
    group, scale = case["heads"] // kv, dim ** -0.5
    first = 0
    for e, (start, n) in enumerate(s["requests"]):
        ctx = start + n
        pages = s["table"][e, :-(-ctx // P)].long()
        k = _values4(*(t[pages] for t in s["keys"])).transpose(1, 2).reshape(-1, kv, dim)[:ctx]
        v = _values4(*(t[pages] for t in s["values"])).transpose(1, 2).reshape(-1, kv, dim)[:ctx]
        q = s["q"][first:first + n].float()
        at = torch.arange(start, ctx, device=DEVICE)[:, None]
        key = torch.arange(ctx, device=DEVICE)[None]
        hidden = key > at
        if case["window"]:
            hidden |= key <= at - case["window"]
        heads = []
        for h in range(kv):
            x = q[:, h * group:(h + 1) * group].transpose(0, 1) @ k[:, h].T.contiguous() * scale
            x.masked_fill_(hidden, -math.inf)
            x = (x - x.amax(-1, keepdim=True)).exp_()
            heads.append((x @ v[:, h] / x.sum(-1, keepdim=True)).transpose(0, 1))
        out.append(torch.cat(heads, 1))
        first += n
    return torch.cat(out).to(TYPES[case["dtype"]])


def _places(requests, table, page):
    """Page and slot of every token of the step."""
    pages, slots = [], []
    for e, (start, n) in enumerate(requests):
        pos = torch.arange(start, start + n, device=DEVICE)
        pages.append(table[e, pos // page].long())
        slots.append(pos % page)
    return torch.cat(pages), torch.cat(slots)


def _plain_store(s):
    where = s["pages"], slice(None), s["slots"]
    out = []
    for x, held in ((s["k"], s["keys"]), (s["v"], s["values"])):
        for t, new in zip(held, _quantize4(x)):
            t[where] = new
        out.append(_values4(*(t[where] for t in held)))
    return [x.to(s["k"].dtype) for x in out]


def _plain_product(s):
    if s["case"]["kind"] == "linear":
        codes, scale = _quantize8(s["x"])
        sums = codes @ s["codes"].double().T
        return (sums.float() * scale[:, None] * s["scale"]).to(s["x"].dtype)
    resid = s["resid"] + s["delta"].float()
    codes, scale = _quantize8(_rms(resid, s["norm"]))
    sums = (codes @ s["codes"].double().T).float() * scale[:, None] * s["scale"]
    gate, up = sums.chunk(2, 1)
    return [(gate / (1 + (-gate).exp()) * up).to(s["delta"].dtype), resid]


# ------------------------------------------------------------------ the framework's


def _ops():
    from tokensprint_amd.kernels import load_hip_ops
    return load_hip_ops(DEVICE)


def _batch(requests, table):
    """The step's description, as the engine hands it to its kernels."""
    from tokensprint_amd.engine.batch import StepBatch
    starts, lens = [r[0] for r in requests], [r[1] for r in requests]

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=DEVICE)

    positions = torch.cat([torch.arange(s, s + n) for s, n in requests]).to(torch.int32)
    q_start = [0]
    for n in lens:
        q_start.append(q_start[-1] + n)
    B, T = len(requests), q_start[-1]
    return StepBatch(
        num_tokens=T, num_entries=B, num_logit_rows=0, token_ids=torch.zeros(T, dtype=torch.int32, device=DEVICE),
        positions=positions.to(DEVICE),
        entry_of_token=ints([e for e, n in enumerate(lens) for _ in range(n)]),
        q_start=ints(q_start), ctx_len=ints([s + n for s, n in requests]), slot_ids=ints(list(range(B))),
        logit_rows=ints([0]), tables=[table], q_lens=lens, starts=starts, max_q_len=max(lens),
        max_ctx_len=max(s + n for s, n in requests))


def _own_cache(case, num_pages):
    from tokensprint_amd.cache import packed_cache
    return packed_cache(num_pages, case["kv_heads"], case["page"], case["dim"], DEVICE)


# ------------------------------------------------------------------ prepare, run


def prepare(case, seed):
    if case["kind"] in ("linear", "gate_up"):
        s = dict(case=case, **_product_inputs(case, seed))
        w = s.pop("w")
        if own:
            return dict(s, ops=_ops(), weight=_ops().quantize_weight(w))
        codes, scale = _quantize8(w)
        return dict(s, codes=codes.to(torch.int8), scale=scale)
    requests, table, held, q = _step_inputs(case, seed)
    s = dict(case=case, requests=requests, table=table, q=q)
    num_pages = int(table.max()) + 1
    if case["kind"] == "store":
        s.update(k=torch.cat([k for k, _ in held]), v=torch.cat([v for _, v in held]))
    if own:
        ops, cache = _ops(), _own_cache(case, num_pages)
        s.update(ops=ops, cache=cache, batch=_batch(requests, table))
        if case["kind"] == "attend":
            for e, (start, n) in enumerate(requests):      # what earlier steps have cached
                before = _batch([(0, start + n)], table[e:e + 1])
                ops.kv_store(*held[e], before, table[e:e + 1], cache)
        return s
    kv, dim, P, n = case["kv_heads"], case["dim"], case["page"], _groups(case["dim"])
    for name in ("keys", "values"):
        s[name] = (torch.zeros(num_pages, kv, P, dim, dtype=torch.uint8, device=DEVICE),
                   torch.zeros(num_pages, kv, P, n, dtype=torch.half, device=DEVICE),
                   torch.zeros(num_pages, kv, P, n, dtype=torch.uint8, device=DEVICE))
    if case["kind"] == "store":
        s["pages"], s["slots"] = _places(requests, table, P)
        return s
    for e, (start, n) in enumerate(requests):
        pages, slots = _places([(0, start + n)], table[e:e + 1], P)
        for x, name in zip(held[e], ("keys", "values")):
            for t, new in zip(s[name], _quantize4(x)):
                t[pages, :, slots] = new
    return s


def run(s):
    case = s["case"]
    if not own:
        return {"attend": _plain_attend, "store": _plain_store, "linear": _plain_product,
                "gate_up": _plain_product}[case["kind"]](s)
    ops = s["ops"]
    if case["kind"] == "attend":
        return ops.paged_attention(
            s["q"], s["batch"], s["table"], s["cache"], num_heads=case["heads"],
            num_kv_heads=case["kv_heads"], head_dim=case["dim"], scale=case["dim"] ** -0.5,
            window=case["window"] or None)
    if case["kind"] == "store":
        ops.kv_store(s["k"], s["v"], s["batch"], s["table"], s["cache"])
        return list(ops.kv_values(s["batch"], s["table"], s["cache"], num_kv_heads=case["kv_heads"],
                                  head_dim=case["dim"], out_dtype=s["k"].dtype))
    if case["kind"] == "linear":
        return ops.linear(s["x"], s["weight"], s["x"].dtype)
    return list(ops.norm_linear(s["resid"], s["delta"], s["norm"], EPS, s["weight"], s["delta"].dtype,
                                silu_mul=True))


# ------------------------------------------------------------------ in 64 bits


def _nearest4(x):
    """What a cache in 4 bits makes of [..., dim], group by group, in 64 bits."""
    out = x.double()
    for a in range(0, x.shape[-1], GROUP):
        part = x[..., a:a + GROUP].double()
        least = torch.minimum(part.min(-1, keepdim=True)[0], torch.zeros((), dtype=torch.double, device=x.device))
        most = torch.maximum(part.max(-1, keepdim=True)[0], torch.zeros((), dtype=torch.double, device=x.device))
        # (a step is a held number: float32's subtraction and division, then float16's rounding)
        way = (most.float() - least.float()).div(torch.full_like(most, 15.0, dtype=torch.float32))
        step = way.clamp(max=65504.0).half().double()
        by = torch.where(step > 0, step, 1.0)
        zero = (-least / by).round().clamp(max=15.0)
        whole = ((part / by).round() + zero).clamp(0, 15) - zero
        out[..., a:a + GROUP] = step * whole
    return out


def _nearest8(x, scale):
    return torch.where(scale > 0, (x / torch.where(scale > 0, scale, 1.0)).round(), 0.0) * scale


def _scale8(x):
    top = torch.maximum(x.max(1, keepdim=True)[0], -x.min(1, keepdim=True)[0]).float()
    return top.div(torch.full_like(top, 127.0)).double()


def exact(case, seed):
    if case["kind"] in ("linear", "gate_up"):
        s = _product_inputs(case, seed)
        w = s["w"].double()
        w = _nearest8(w, _scale8(w))
        if case["kind"] == "linear":
            x = s["x"].double()
            return _nearest8(x, _scale8(x)) @ w.T
        resid = s["resid"].double() + s["delta"].double()
        h = resid / ((resid ** 2).sum(1, keepdim=True) / case["K"] + EPS).sqrt() * s["norm"].double()
        y = _nearest8(h, _scale8(h)) @ w.T
        gate, up = y[:, :case["N"]], y[:, case["N"]:]
        return [gate * torch.sigmoid(gate) * up, resid]
    requests, _, held, q = _step_inputs(case, seed)
    if case["kind"] == "store":
        return [_nearest4(torch.cat([pair[i] for pair in held])) for i in (0, 1)]
    per, out, first = case["heads"] // case["kv_heads"], [], 0
    for (start, n), (k, v) in zip(requests, held):
        k, v = _nearest4(k), _nearest4(v)
        rows = q[first:first + n].double()
        o = torch.empty_like(rows)
        for i in range(0, n, 512):                  # so many queries at a time
            m = min(512, n - i)
            pos = start + i + torch.arange(m, device=DEVICE)
            near = torch.arange(start + n, device=DEVICE)
            far = pos[:, None] - near[None]
            seen = (far >= 0) & (far < (case["window"] or start + n))
            for h in range(case["heads"]):
                score = rows[i:i + m, h] @ k[:, h // per].T / math.sqrt(case["dim"])
                o[i:i + m, h] = torch.softmax(score.masked_fill(~seen, -math.inf), 1) @ v[:, h // per]
        out.append(o)
        first += n
    return torch.cat(out)

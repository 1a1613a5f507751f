"""The operators of a decoder block held in few bits, and how fast they run.

  linear_i8  the Linear node over 8-bit weights: rows of X are rounded to 8-bit
             integers with a scale each, the product is summed in 32-bit
             integers, and the scales of row and output channel, the bias, the
             activation and the residual follow.
  norm_rope  between the fused query / key / value projection and attention:
             RMS norm of every query and key head, the position rotation, and
             the step from token-major rows to the head-major planes that
             attention reads.
  attention_q4  attention over a KV cache held in 4 bits (groups of 32 values
             of a row, each with a scale and a minimum): the call's new rows
             are rounded and appended, and every key is attended as stored.

`own` false computes them in elementary torch operations; true makes the calls
a Python host makes of libvai_amd.so.
"""
import ctypes
import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16}
BYTES = {"f32": 4, "f16": 2}
GROUP = 32   # values of a cached row that share a scale and a minimum


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # One token through a large-model up projection: bound by reading the weight once.
        _linear("i8_decode_m1", 1, 2048, 8192),
        # A few sequences decoded together, in the engine's default fp32 between nodes.
        _linear("i8_decode_m7_f32", 7, 4096, 5120, x="f32", out="f32", bias=True),
        # A short prompt of odd length through odd widths, with activation.
        _linear("i8_prompt_m61_odd", 61, 1999, 5003, bias=True, act="GELU_TANH"),
        # A prompt through an attention output projection with its residual.
        _linear("i8_prompt_m500", 500, 2048, 2048, x="f32", out="f32", residual=True),
        # A long prompt's gate and up projection: the largest product.
        _linear("i8_prefill_m2048", 2048, 4096, 16384),
        # One token's heads on their way to the cache: launch latency.
        _norm_rope("norm_rope_decode", 1, 1, 32, 8, 64, count=3000),
        # Two prompts of odd length, odd head size, a part of each head rotated in neighbouring pairs.
        _norm_rope("norm_rope_t333_odd", 2, 333, 12, 4, 80, rot=40, pairs="neighbours", count=17, x="f32", out="f32"),
        # A long prompt's heads at far positions: one pass over the projection.
        _norm_rope("norm_rope_t4096", 1, 4096, 32, 8, 128, count=100000),
        # One token against a KV cache: the attention of every decode step.
        _attention("q4_decode_cache", 32, 8, 64, 1, 4096, 3000),
        # One token against a very long cache: bound by reading the cache once.
        _attention("q4_decode_long", 32, 8, 128, 1, 131072, 120001),
        # Five drafted tokens checked at once over a sliding window in a ring, large heads.
        _attention("q4_draft5_ring", 8, 2, 256, 5, 4352, 70000, ring=True, span=4096),
        # A chunk of a prompt over what is cached already.
        _attention("q4_chunk_t512", 32, 8, 128, 512, 8192, 7001),
    ]


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    kind = rng.choice(("decode", "decode", "prompt", "prompt", "prefill", "heads", "heads", "heads",
                       "token", "token", "draft", "chunk", "chunk"))
    if kind in ("decode", "prompt", "prefill"):
        lo, hi = {"decode": (1, 16), "prompt": (17, 700), "prefill": (700, 4096)}[kind]
        k, n, m = _size(rng, 64, 11008), _size(rng, 64, 16384), _log(rng, lo, hi)
        while m * k * n > 2048 * 4096 * 16384 or n * k + 4 * m * k + 8 * m * n > 150000000:
            k, n = max(64, k * 3 // 4), max(64, n * 3 // 4)
        return _linear(None, m, k, n, x=rng.choice(("f16", "f16", "f32")), out=rng.choice(("f16", "f32")),
                       bias=rng.random() < 0.5, residual=rng.random() < 0.3,
                       act=rng.choice(("NONE", "NONE", "GELU_TANH", "SILU")))
    if kind == "heads":
        hkv = rng.choice((1, 2, 4, 8, 12))
        hq, d = hkv * rng.choice((1, 2, 3, 4)), rng.choice((32, 64, 64, 72, 80, 96, 128, 128, 256))
        batch, t = rng.choice((1, 1, 1, 2, 5)), _log(rng, 1, 4096)
        while batch * t * (hq + 2 * hkv) * d > 4096 * 48 * 64:
            t = (t + 1) // 2
        return _norm_rope(None, batch, t, hq, hkv, d, rot=rng.choice((d, d, d // 2)),
                          pairs=rng.choice(("halves", "halves", "neighbours")), norm=rng.random() < 0.8,
                          count=_log(rng, 1, 1000000) - 1, x=rng.choice(("f16", "f16", "f32")),
                          out=rng.choice(("f16", "f16", "f32")))
    hkv, d = rng.choice((1, 2, 4, 8, 12)), rng.choice((32, 64, 64, 80, 96, 128, 128, 256))
    hq = hkv * rng.choice((1, 2, 4, 5, 8))
    ring, x = rng.random() < 0.25, rng.choice(("f16", "f16", "f32"))
    if kind == "chunk":
        t, cache = _log(rng, 17, 1500), 256 * _log(rng, 1, 32)
        t = min(t, cache)
        while hq * d * t * cache > 32 * 128 * 512 * 8192:
            t = (t + 1) // 2
        if t >= cache:
            ring = False
    else:
        t, cache = 1 if kind == "token" else rng.randint(2, 16), 256 * _log(rng, 1, 512)
        while hkv * d * cache > 8 * 128 * 131072:
            cache = 256 * max(1, cache // 512)
    count = _log(rng, 1, 2 * cache) if ring else _log(rng, 1, cache - t + 1) - 1
    span = rng.randint(1, cache - t + 1) if ring else rng.choice((0, 0, 0, 512))
    return _attention(None, hq, hkv, d, t, cache, count, ring=ring, span=span, x=x)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A layer width: mostly a multiple of 128 or 64, sometimes of 8, sometimes odd."""
    n = _log(rng, lo, hi)
    step = rng.choice((128, 128, 128, 64, 64, 8, 1))
    return max(lo, n // step * step)


def _named(name, case):
    return dict(case, name=name) if name else case


def _linear(name, m, k, n, x="f16", out="f16", bias=False, residual=False, act="NONE"):
    return _named(name, {"op": "linear_i8", "m": m, "k": k, "n": n, "x": x, "out": out, "bias": bias,
                         "residual": residual, "act": act})


def _norm_rope(name, batch, t, hq, hkv, d, rot=None, pairs="halves", norm=True, count=0, x="f16", out="f16"):
    return _named(name, {"op": "norm_rope", "batch": batch, "t": t, "hq": hq, "hkv": hkv, "d": d, "rot": rot or d,
                         "pairs": pairs, "norm": norm, "count": count, "x": x, "out": out})


def _attention(name, hq, hkv, d, t, cache, count, ring=False, span=0, x="f16", out="f16"):
    return _named(name, {"op": "attention_q4", "hq": hq, "hkv": hkv, "d": d, "t": t, "cache": cache, "count": count,
                         "ring": ring, "span": span, "x": x, "out": out})


THETA, EPS = 500000.0, 1e-5


# ---- inputs ------------------------------------------------------------------

class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, shape, dtype, sigma=1.0):
        if dtype == "f16":
            return torch.randn(shape, generator=self.g, device="cuda", dtype=torch.float16).mul_(sigma)
        return torch.randn(shape, generator=self.g, device="cuda").mul_(sigma)


def _first(c):
    """The oldest position a cached call finds: a ring holds the last `cache` ones, the call's own among them."""
    return max(0, c["count"] + c["t"] - c["cache"]) if c["ring"] else 0


def _inputs(case, seed):
    """The tensors of a case from its seed: what both prepare() and exact() start from."""
    r, c = _Rand(seed), case
    if c["op"] == "linear_i8":
        w = r.normal((c["n"], c["k"]), "f32", 0.02)
        scale = w.abs().amax(1) / 127
        t = {"w": torch.round(w / scale[:, None]).to(torch.int8), "w_scale": scale,
             "x": r.normal((c["m"], c["k"]), c["x"])}
        if c["bias"]:
            t["bias"] = r.normal((c["n"],), "f32", 0.02)
        if c["residual"]:
            t["residual"] = r.normal((c["m"], c["n"]), c["out"])
        return t
    if c["op"] == "norm_rope":
        heads = c["hq"] + 2 * c["hkv"]
        t = {"qkv": r.normal((c["batch"], c["t"], heads * c["d"]), c["x"], 2.0)}
        if c["norm"]:
            t["q_weight"] = r.normal((c["d"],), "f16", 0.1) + 1
            t["k_weight"] = r.normal((c["d"],), "f16", 0.1) + 1
        return t
    old = c["count"] - _first(c)
    # keys have channels that stand out, as projections give them; values do not
    loud = 1 + 4 * (torch.rand((c["hkv"], 1, c["d"]), generator=r.g, device="cuda") > 0.95)
    t = {"q": r.normal((c["hq"], c["t"], c["d"]), c["x"])}
    for name, n in (("old", old), ("new", c["t"])):
        t["k_" + name] = r.normal((c["hkv"], n, c["d"]), c["x"]).mul_(loud.to(TORCH[c["x"]]))
        t["v_" + name] = r.normal((c["hkv"], n, c["d"]), c["x"])
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:
        return _own_prepare(case, t)
    if case["op"] == "attention_q4":     # the cache as a program without 4-bit storage of its own would keep it
        for name in ("k", "v"):
            codes, scale, low = _round4(t.pop(f"{name}_old"))
            room = lambda x: torch.cat((x, x.new_zeros((x.shape[0], case["t"]) + x.shape[2:])), 1)  # noqa: E731
            t[name] = tuple(room(x) for x in (codes, scale, low))
    return {"case": case, "t": t}


def run(state):
    if own:
        return _own_run(state)
    return {"linear_i8": _plain_linear, "norm_rope": _plain_norm_rope,
            "attention_q4": _plain_attention}[state["case"]["op"]](state["case"], state["t"])


# ---- the plain forms ----------------------------------------------------------

def _act(x, name):
    if name == "SILU":
        return x / (1 + torch.exp(-x))
    if name == "GELU_TANH":
        return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return x


def _plain_linear(c, t):
    x = t["x"].float()
    # (divided in 64 bits: the scale, and a quotient next to a half, must round as they stand)
    scale = (x.abs().amax(1, keepdim=True).double() / 127).float()
    codes = torch.round(x.double() / scale.double()).float()
    acc = torch.zeros((c["m"], c["n"]), dtype=torch.float64, device="cuda")
    for k in range(0, c["k"], 1024):     # 1024 products of 8-bit integers sum exactly in fp32
        acc += codes[:, k:k + 1024] @ t["w"][:, k:k + 1024].float().t()
    y = acc.float() * scale * t["w_scale"]
    if c["bias"]:
        y = y + t["bias"]
    y = _act(y, c["act"])
    if c["residual"]:
        y = y + t["residual"].float()
    return y.to(TORCH[c["out"]])


def _plain_norm_rope(c, t):
    b, n, hq, hkv, d, rot = c["batch"], c["t"], c["hq"], c["hkv"], c["d"], c["rot"]
    x = t["qkv"].float().view(b, n, hq + 2 * hkv, d).transpose(1, 2)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if c["norm"]:
        q, k = (y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * t[w].float()
                for y, w in ((q, "q_weight"), (k, "k_weight")))
    # (angles in 64 bits: at a far position fp32 holds too little of them)
    freq = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = (torch.arange(n, dtype=torch.float64, device="cuda") + c["count"])[:, None] * freq
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def turn(y):
        r, rest = y[..., :rot], y[..., rot:]
        if c["pairs"] == "halves":
            a, e = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat((a * cos - e * sin, e * cos + a * sin), -1)
        else:
            a, e = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - e * sin, e * cos + a * sin), -1).flatten(-2)
        return torch.cat((r, rest), -1)

    return tuple(y.to(TORCH[c["out"]]).contiguous() for y in (turn(q), turn(k), v))


def _round4(x):
    """fp16 rows to 4-bit codes with a scale and a minimum for each group of 32 (a last group may be shorter)."""
    x = x.half().float()
    codes, scales, lows = [], [], []
    for g in range(0, x.shape[-1], GROUP):
        y = x[..., g:g + GROUP]
        low = y.amin(-1, keepdim=True)
        scale = ((y.amax(-1, keepdim=True) - low).double() / 15).half()
        n = torch.round((y - low).double() / scale.double())     # (0 / 0 where a group is constant)
        codes.append(torch.nan_to_num(n, 0.0).clamp_(0, 15).to(torch.uint8))
        scales.append(scale)
        lows.append(low.half())
    return torch.cat(codes, -1), torch.cat(scales, -1), torch.cat(lows, -1)


def _value4(codes, scale, low):
    spread = lambda x: x.float().repeat_interleave(GROUP, -1)[..., :codes.shape[-1]]  # noqa: E731
    return codes.float() * spread(scale) + spread(low)


def _plain_attention(c, t):
    hkv, group, n, first = c["hkv"], c["hq"] // c["hkv"], c["t"], _first(c)
    pos = torch.arange(n, device="cuda")[:, None] + c["count"]
    key = torch.arange(first, c["count"] + n, device="cuda")[None, :]
    see = key <= pos
    if c["span"]:
        see = see & (key > pos - c["span"])
    rows = []
    for name in ("k", "v"):
        for kept, new in zip(t[name], _round4(t[name + "_new"])):
            kept[:, -n:] = new
    out = torch.empty((n, c["hq"], c["d"]), device="cuda")
    q = t["q"].float().view(hkv, group, n, c["d"])
    for h in range(hkv):
        k, v = (_value4(*(x[h] for x in t[name])) for name in ("k", "v"))
        s = (q[h].reshape(group * n, -1) @ k.t() / math.sqrt(c["d"])).view(group, n, -1)
        s = s.masked_fill(~see, -math.inf)
        e = torch.exp(s - s.amax(-1, keepdim=True))
        o = e.view(group * n, -1) @ v / e.sum(-1).view(group * n, 1)
        out[:, h * group:(h + 1) * group] = o.view(group, n, -1).transpose(0, 1)
        rows.append((k[-n:], v[-n:]))
    return out.to(TORCH[c["out"]]), torch.stack([r[0] for r in rows]), torch.stack([r[1] for r in rows])


# ---- the framework's calls ----------------------------------------------------

class _Dev:
    """A torch tensor as the buffer handle _capi's argument builders take."""

    def __init__(self, t, code=None, shape=None):
        from vai_amd import _capi as capi
        self.t, self.ptr, self.shape = t, t.data_ptr(), tuple(shape or t.shape)
        self.nbytes = t.numel() * t.element_size()
        self.code = {torch.float32: capi.F32, torch.float16: capi.F16}.get(t.dtype) if code is None else code


def _workspace(a, need):
    if not need:
        return None
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    return ws


def _own_prepare(c, t):
    from vai_amd import _capi as capi
    L, stream = capi.lib(), torch.cuda.current_stream().cuda_stream
    dev = lambda name: _Dev(t[name]) if name in t else None  # noqa: E731
    if c["op"] == "linear_i8":
        out = torch.empty((c["m"], c["n"]), dtype=TORCH[c["out"]], device="cuda")
        # 8-bit rows start on 16-byte boundaries
        w = torch.zeros((c["n"], capi.i8_stride(c["k"])), dtype=torch.int8, device="cuda")
        w[:, :c["k"]] = t.pop("w")
        a = capi.linear_i8_args(_Dev(out), dev("x"), _Dev(w), dev("w_scale"), dev("bias"), dev("residual"),
                                epi=c["act"])
        a.bias_repeat = c["n"] if c["bias"] else 0
        ws = _workspace(a, L.vai_linear_i8_workspace_size(ctypes.byref(a)))
        return {"calls": ((L.vai_linear_i8_launch, (ctypes.byref(a), stream)),), "out": out, "keep": (a, ws, w, t)}
    if c["op"] == "norm_rope":
        q, k, v = (torch.empty((c["batch"], h, c["t"], c["d"]), dtype=TORCH[c["out"]], device="cuda")
                   for h in (c["hq"], c["hkv"], c["hkv"]))
        count = torch.tensor([c["count"]], dtype=torch.int32, device="cuda")
        a = capi.qk_norm_rope_args(_Dev(q), _Dev(k), _Dev(v), dev("qkv"), dev("q_weight"), dev("k_weight"),
                                   norm=c["norm"], eps=EPS, theta=THETA, rot_dim=c["rot"],
                                   pairs={"halves": "HALVES", "neighbours": "NEIGHBOURS"}[c["pairs"]],
                                   count=_Dev(count))
        return {"calls": ((L.vai_qk_norm_rope_launch, (ctypes.byref(a), stream)),), "out": (q, k, v),
                "keep": (a, count, t)}
    hkv, d, n, first = c["hkv"], c["d"], c["t"], _first(c)
    size = capi.attention_cache_bytes(hkv, c["cache"], d, capi.Q4)
    kc, vc = (torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(2))
    planes = [_Dev(x, capi.Q4, (hkv, c["cache"], d)) for x in (kc, vc)]
    count = torch.tensor([first], dtype=torch.int32, device="cuda")
    k_old, v_old = t.pop("k_old"), t.pop("v_old")
    if k_old.shape[1]:                   # what is cached already: appended as a prompt is
        scrap = torch.empty((1, 1, c["hq"], d), dtype=torch.float16, device="cuda")
        a = capi.attention_args(_Dev(scrap), _Dev(t["q"][None, :, :1].contiguous()), _Dev(k_old[None]), _Dev(v_old[None]),
                                causal=True, span=1, cache=(*planes, _Dev(count), c["ring"]))
        ws = _workspace(a, L.vai_attention_workspace_size(ctypes.byref(a)))
        capi.check(L.vai_attention_launch(ctypes.byref(a), stream), "append")
        torch.cuda.synchronize()
        del ws
    count.fill_(c["count"])
    out = torch.empty((1, n, c["hq"], d), dtype=TORCH[c["out"]], device="cuda")
    a = capi.attention_args(_Dev(out), _Dev(t["q"][None]), _Dev(t["k_new"][None]), _Dev(t["v_new"][None]), causal=True,
                            span=c["span"], cache=(*planes, _Dev(count), c["ring"]))
    ws = _workspace(a, L.vai_attention_workspace_size(ctypes.byref(a)))
    rows = [torch.empty((hkv, n, d), dtype=torch.float32, device="cuda") for _ in range(2)]
    read = capi.attention_cache_read_args(*(_Dev(x) for x in rows), *planes, c["count"] % c["cache"])
    return {"calls": ((L.vai_attention_launch, (ctypes.byref(a), stream)),
                      (L.vai_attention_cache_read, (ctypes.byref(read), stream))),
            "out": (out[0], *rows), "keep": (a, read, ws, kc, vc, count, t)}


def _own_run(state):
    for call, args in state["calls"]:
        status = call(*args)
        if status:
            from vai_amd import _capi as capi
            capi.check(status, "launch")
    return state["out"]


# ---- work and 64-bit results ----------------------------------------------------

def work(case):
    c = case
    if c["op"] == "linear_i8":
        m, k, n = c["m"], c["k"], c["n"]
        bytes_ = n * k + 4 * n * (2 if c["bias"] else 1) + m * k * BYTES[c["x"]]
        return {"bytes": bytes_ + m * n * BYTES[c["out"]] * (2 if c["residual"] else 1), "flops": 2 * m * n * k}
    if c["op"] == "norm_rope":
        moved = c["batch"] * c["t"] * (c["hq"] + 2 * c["hkv"]) * c["d"]
        turned = c["batch"] * c["t"] * (c["hq"] + c["hkv"]) * c["d"]
        return {"bytes": moved * (BYTES[c["x"]] + BYTES[c["out"]]) + (4 * c["d"] if c["norm"] else 0),
                "flops": turned * (3 + (4 if c["norm"] else 0))}
    pairs, low = 0, c["count"]
    for i in range(c["t"]):
        pos = c["count"] + i
        beg = max(0, pos + 1 - c["span"]) if c["span"] else 0
        pairs, low = pairs + pos + 1 - beg, min(low, beg)
    row = c["d"] / 2 + 4 * math.ceil(c["d"] / GROUP)
    new = 2 * c["t"] * c["hkv"]
    bytes_ = c["t"] * c["hq"] * c["d"] * (BYTES[c["x"]] + BYTES[c["out"]]) + 2 * (c["count"] - low) * c["hkv"] * row
    return {"bytes": bytes_ + new * (c["d"] * BYTES[c["x"]] + row + 4 * c["d"]), "flops": 4 * c["d"] * c["hq"] * pairs}


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    if c["op"] == "linear_i8":
        x = t["x"].double()
        step = (x.abs().max(1).values / 127).float().double()       # the scale is kept as fp32
        y = torch.round(x / step[:, None]) @ t["w"].double().t()
        y = y * step[:, None] * t["w_scale"].double()[None, :]
        if "bias" in t:
            y = y + t["bias"].double()
        if c["act"] == "SILU":
            y = y * torch.sigmoid(y)
        elif c["act"] == "GELU_TANH":
            y = y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
        return y + t["residual"].double() if "residual" in t else y
    if c["op"] == "norm_rope":
        b, n, d, half = c["batch"], c["t"], c["d"], c["rot"] // 2
        x = t["qkv"].double().view(b, n, -1, d)
        q, k, v = x.split((c["hq"], c["hkv"], c["hkv"]), 2)
        if c["norm"]:
            q = q * (q.square().sum(-1, keepdim=True) / d + EPS).rsqrt() * t["q_weight"].double()
            k = k * (k.square().sum(-1, keepdim=True) / d + EPS).rsqrt() * t["k_weight"].double()
        # each pair as a complex number, turned by its angle
        i = torch.arange(half, device="cuda", dtype=torch.float64)
        pos = torch.arange(c["count"], c["count"] + n, device="cuda", dtype=torch.float64)
        unit = torch.polar(torch.ones((n, half), dtype=torch.float64, device="cuda"),
                           pos[:, None] * torch.exp(-i * math.log(THETA) / half))[None, :, None, :]
        lo = torch.arange(half, device="cuda") * (1 if c["pairs"] == "halves" else 2)
        hi = lo + (half if c["pairs"] == "halves" else 1)
        for y in (q, k):
            z = torch.complex(y[..., lo], y[..., hi]) * unit
            y[..., lo], y[..., hi] = z.real, z.imag
        return tuple(y.permute(0, 2, 1, 3).contiguous() for y in (q, k, v))
    n, group, first = c["t"], c["hq"] // c["hkv"], _first(c)
    kept = {}
    for name in ("k", "v"):
        x = torch.cat((t.pop(f"{name}_old"), t[f"{name}_new"]), 1).half().double()
        for g in range(0, c["d"], GROUP):
            y = x[..., g:g + GROUP]
            low, high = y.min(-1).values[..., None], y.max(-1).values[..., None]
            step = ((high - low) / 15).half().double()
            level = torch.where(step > 0, torch.round((y - low) / step), torch.zeros_like(y)).clamp(0, 15)
            x[..., g:g + GROUP] = level * step + low
        kept[name] = x
    key = torch.arange(first, c["count"] + n, device="cuda")
    out = torch.empty((n, c["hq"], c["d"]), dtype=torch.float64, device="cuda")
    for h in range(c["hq"]):
        s = t["q"][h].double() @ kept["k"][h // group].t() / math.sqrt(c["d"])
        pos = torch.arange(c["count"], c["count"] + n, device="cuda")[:, None]
        hide = (key > pos) | (key <= pos - c["span"]) if c["span"] else key > pos
        out[:, h] = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ kept["v"][h // group]
    return out, kept["k"][:, -n:].contiguous(), kept["v"][:, -n:].contiguous()

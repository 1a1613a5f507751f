"""Serving many sequences from a KV cache in pages, and how fast its operators run.

  append     from the fused query / key / value projection of a ragged batch: the
             RMS norm of query and key heads, the position rotation, queries to
             token-major rows, keys and values into the pages of their sequence.
  attention  the new tokens of every sequence (one each, a few drafted ones, a
             chunk of a prompt) over the pages that the sequence holds.
  verify     drafted tokens against the target's probabilities: which are kept,
             and the token that follows, from given random numbers.

`own` false computes them in elementary torch operations; true makes the calls
a Python host makes of libvai_amd.so.
"""
import ctypes
import math
import random

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16}
BYTES = {"f32": 4, "f16": 2}
THETA, EPS = 500000.0, 1e-5


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # One sequence's next token on its way to the cache: launch latency.
        _append("append_token", 1, 1, 32, 8, 64, ctx=3000),
        # A few sequences with drafted tokens, odd head size, a part of each head
        # rotated in neighbouring pairs, no norm, rows of padding behind the batch.
        _append("append_drafts_odd", 13, 7, 12, 4, 80, ctx=40000, page=24, ragged=True, pad=5, rot=40,
                pairs="neighbours", norm=False, x="f32", out="f32"),
        # Three prompts packed into one batch: one pass over the projection.
        _append("append_prompts", 3, 1366, 32, 8, 128, ctx=1, page=64, ragged=True),
        # One short conversation's next token: latency.
        _attention("attn_token", 1, 1, 32, 8, 64, ctx=500),
        # A serving step: 64 conversations of very different lengths, a token each.
        _attention("attn_batch64", 64, 1, 32, 8, 128, ctx=8192, ragged=True),
        # One token against a very long context: bound by reading the cache once.
        _attention("attn_long", 1, 1, 32, 8, 128, ctx=131071, page=64),
        # Drafted tokens of several sequences over a sliding window, in the engine's
        # default fp32 between nodes.
        _attention("attn_drafts_span_f32", 7, 6, 40, 8, 64, ctx=20000, page=32, ragged=True, span=4096, x="f32", out="f32"),
        # fp32 pages of an odd size and heads of an odd one.
        _attention("attn_f32_pages_odd", 5, 3, 9, 3, 50, ctx=700, page=24, ragged=True, x="f32", out="f32", pages="f32"),
        # A chunk of one prompt beside the next tokens of other sequences.
        _attention("attn_chunk_mixed", 9, 1, 32, 8, 128, ctx=7001, page=64, ragged=True, chunk=512),
        # One sequence's greedy drafts from a lookup (no probabilities of their own).
        _verify("verify_greedy", 1, 4, 32768, draft="none", temp="greedy"),
        # A batch of drafts, sampled, odd vocabulary, some sequences greedy.
        _verify("verify_mixed_odd", 5, 5, 50021, ragged=True, temp="mixed"),
        # A large vocabulary in fp32, many sequences: one pass over both models' logits.
        _verify("verify_batch32", 32, 5, 131072, x="f32"),
    ]


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    kind = rng.choice(("append", "append", "append", "token", "token", "drafts", "drafts", "chunk", "verify", "verify"))
    mix = rng.randrange(1 << 30)
    if kind == "verify":
        vocab = _log(rng, 1000, 160000)
        vocab = vocab // rng.choice((1, 8, 64)) * 64 if vocab > 4096 and rng.random() < 0.5 else vocab
        batch, drafts = _log(rng, 1, 64), rng.randint(0, 8)
        while batch * (drafts + 1) * vocab > 32 * 6 * 131072:
            batch = (batch + 1) // 2 if batch > 1 else 1
            drafts = drafts if batch > 1 else drafts - 1
        return _verify(None, batch, drafts, min(vocab, 160000), ragged=rng.random() < 0.6,
                       temp=rng.choice(("sampled", "sampled", "mixed", "greedy")),
                       draft=rng.choice(("logits", "logits", "none")), x=rng.choice(("f16", "f32")), mix=mix)
    hkv, d = rng.choice((1, 2, 4, 8, 12)), rng.choice((32, 50, 64, 64, 72, 80, 96, 128, 128, 128, 256))
    hq = hkv * rng.choice((1, 2, 3, 4, 5, 8))
    page = rng.choice((8, 16, 16, 16, 24, 32, 64, 64, 128, 256))
    ragged, pad = rng.random() < 0.7, rng.choice((0, 0, 3))
    if kind == "append":
        batch, new = _log(rng, 1, 64), _log(rng, 1, 4096)
        while batch * new * (hq + 2 * hkv) * d > 4098 * 48 * 128:
            batch, new = (batch + 1) // 2, (new + 1) // 2 if batch == 1 or new > 64 else new
        return _append(None, batch, new, hq, hkv, d, ctx=_log(rng, 1, 200000) - 1, page=page, ragged=ragged, pad=pad,
                       rot=rng.choice((d, d, d // 4 * 2)), pairs=rng.choice(("halves", "halves", "neighbours")),
                       norm=rng.random() < 0.7, x=rng.choice(("f16", "f16", "f32")), out=rng.choice(("f16", "f16", "f32")),
                       pages=rng.choice(("f16", "f16", "f16", "f32")), mix=mix)
    x = rng.choice(("f16", "f16", "f32"))
    out = rng.choice((x, x, "f16"))
    if kind == "chunk":
        chunk, batch, new = _log(rng, 17, 2048), _log(rng, 1, 16), rng.choice((1, 1, 4))
        ctx = _log(rng, 1, 16384)
        while hq * d * chunk * (ctx + chunk / 2) > 32 * 128 * 512 * 7257:
            chunk, ctx = (chunk + 1) // 2, (ctx + 1) // 2
        pages = "f16"
    else:
        chunk, batch, new = 0, _log(rng, 1, 128), 1 if kind == "token" else rng.randint(2, 8)
        ctx, pages = _log(rng, 1, 131071), rng.choice(("f16", "f16", "f16", "f32"))
    while batch * (ctx + new) * hkv * d * (2 if pages == "f32" else 1) > 64 * 2048 * 8 * 128:
        if batch > 1 and (batch > 16 or rng.random() < 0.5):
            batch //= 2
        else:
            ctx = max(1, ctx // 2)
    return _attention(None, batch, new, hq, hkv, d, ctx=ctx, page=page, ragged=ragged, pad=pad, chunk=chunk,
                      span=rng.choice((0, 0, 0, rng.randint(1, 5000))), x=x, out=out, pages=pages, mix=mix)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _named(name, case):
    return dict(case, name=name) if name else case


def _append(name, batch, new, hq, hkv, d, ctx, page=16, ragged=False, pad=0, rot=None, pairs="halves", norm=True,
            x="f16", out="f16", pages="f16", mix=1):
    return _named(name, {"op": "append", "batch": batch, "new": new, "chunk": 0, "hq": hq, "hkv": hkv, "d": d,
                         "ctx": ctx, "page": page, "ragged": ragged, "pad": pad, "rot": rot or d, "pairs": pairs,
                         "norm": norm, "x": x, "out": out, "pages": pages, "mix": mix})


def _attention(name, batch, new, hq, hkv, d, ctx, page=16, ragged=False, pad=0, chunk=0, span=0, x="f16", out="f16",
               pages="f16", mix=1):
    return _named(name, {"op": "attention", "batch": batch, "new": new, "chunk": chunk, "hq": hq, "hkv": hkv, "d": d,
                         "ctx": ctx, "page": page, "ragged": ragged, "pad": pad, "span": span, "x": x, "out": out,
                         "pages": pages, "mix": mix})


def _verify(name, batch, drafts, vocab, ragged=False, draft="logits", temp="sampled", x="f16", mix=1):
    return _named(name, {"op": "verify", "batch": batch, "drafts": drafts, "vocab": vocab, "ragged": ragged,
                         "draft": draft, "temp": temp, "x": x, "mix": mix})


def _plan(c):
    """(new tokens, positions held before) of each sequence of a case: its raggedness comes from the case alone."""
    r = random.Random(c["mix"])
    if c["op"] == "verify":
        return [(r.randint(0, c["drafts"]) if c["ragged"] else c["drafts"]) + 1 for _ in range(c["batch"])], None
    new = [r.randint(1, c["new"]) if c["ragged"] else c["new"] for _ in range(c["batch"])]
    held = [_log(r, max(1, c["ctx"] // 128), max(1, c["ctx"])) if c["ragged"] else c["ctx"] for _ in range(c["batch"])]
    if c["op"] == "append" and c["ragged"] and c["new"] > 64:    # packed prompts fill the batch
        new = [c["new"] + (i % 3 - 1) * (c["new"] // 5) for i in range(c["batch"])]
    if c["chunk"]:
        new[0], held[0] = c["chunk"], c["ctx"]
    return new, held


# ---- inputs ------------------------------------------------------------------

class _Rand:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, shape, dtype, sigma=1.0):
        if dtype == "f16":
            return torch.randn(shape, generator=self.g, device="cuda", dtype=torch.float16).mul_(sigma)
        return torch.randn(shape, generator=self.g, device="cuda").mul_(sigma)

    def uniform(self, shape):
        return torch.rand(shape, generator=self.g, device="cuda")


def _starts(new):
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return starts


def _inputs(case, seed):
    """The tensors of a case from its seed: what both prepare() and exact() start from."""
    r, c = _Rand(seed), case
    new, held = _plan(c)
    starts = _starts(new)
    t = {"seq_start": torch.tensor(starts, dtype=torch.int32, device="cuda")}
    if c["op"] == "verify":
        rows, v = starts[-1], c["vocab"]
        # a few hundred tokens carry most of a row, as a language model's do; the
        # draft model's logits follow the target's at a distance
        t["target"] = r.normal((rows, v), c["x"], 2.5)
        chosen = t["target"].float()
        if c["draft"] == "logits":
            t["draft"] = (t["target"].float() + r.normal((rows, v), "f32", 0.7)).to(TORCH[c["x"]])
            chosen = t["draft"].float()
        temp = {"greedy": [0.0], "sampled": [0.8], "mixed": [0.7, 0.0, 1.0]}[c["temp"]]
        t["temperature"] = torch.tensor([temp[i % len(temp)] for i in range(c["batch"])], device="cuda")
        # row i's distribution draws the token fed at row i + 1: a greedy sequence's
        # draft model its largest, a lookup mostly the target's largest
        least = 0.1 if c["draft"] == "none" else 0.0
        sharp = t["temperature"].repeat_interleave(torch.tensor(new, device="cuda"))[:, None]
        noise = -torch.log(-torch.log(r.uniform((rows, v)).clamp_(1e-20, 1 - 1e-7)))
        drawn = (chosen + torch.where(sharp > 0, sharp, least) * noise).argmax(-1).to(torch.int32)
        first = r.uniform((rows,)).mul_(v).to(torch.int32)
        t["tokens"] = torch.cat((first[:1], drawn[:-1]))
        t["uniform"] = r.uniform((rows,))
        t["counts"] = (r.uniform((c["batch"],)) * 5000).to(torch.int32)
        return t
    rows, d, hkv, page = starts[-1] + c["pad"], c["d"], c["hkv"], c["page"]
    used = [(h + n + page - 1) // page for h, n in zip(held, new)]
    # a program allots an append's pages only (the positions before it are not read): the table's others are unset
    first = [h // page if c["op"] == "append" else 0 for h in held]
    total = sum(u - f for u, f in zip(used, first)) + 2
    order = torch.randperm(total, generator=r.g, device="cuda").to(torch.int32)
    table = torch.full((c["batch"], max(used) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, (u, f) in enumerate(zip(used, first)):
        table[s, f:u] = order[at:at + u - f]
        at += u - f
    t["table"] = table
    t["counts"] = torch.tensor(held, dtype=torch.int32, device="cuda")
    shape = (total, hkv, page, d)
    if c["op"] == "append":
        t["qkv"] = r.normal((rows, (c["hq"] + 2 * hkv) * d), c["x"], 2.0)
        t["k_pages"], t["v_pages"] = (r.normal(shape, c["pages"]) for _ in range(2))
        if c["norm"]:
            t["q_weight"] = r.normal((d,), "f16", 0.1) + 1
            t["k_weight"] = r.normal((d,), "f16", 0.1) + 1
        return t
    # keys have channels that stand out, as projections give them; values do not
    loud = 1 + 4 * (r.uniform((1, hkv, 1, d)) > 0.95)
    t["q"] = r.normal((rows, c["hq"], d), c["x"])
    t["k_pages"] = r.normal(shape, c["pages"]).mul_(loud.to(TORCH[c["pages"]]))
    t["v_pages"] = r.normal(shape, c["pages"])
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    if own:
        return _own_prepare(case, t)
    return {"case": case, "t": t}


def run(state):
    if own:
        return _own_run(state)
    return {"append": _plain_append, "attention": _plain_attention,
            "verify": _plain_verify}[state["case"]["op"]](state["case"], state["t"])


# ---- the plain forms ----------------------------------------------------------

def _plain_append(c, t):
    new, held = _plan(c)
    n, hq, hkv, d, rot, page = sum(new), c["hq"], c["hkv"], c["d"], c["rot"], c["page"]
    x = t["qkv"][:n].float().view(n, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if c["norm"]:
        q, k = (y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * t[w].float()
                for y, w in ((q, "q_weight"), (k, "k_weight")))
    lens = (t["seq_start"][1:] - t["seq_start"][:-1]).long()
    seq = torch.repeat_interleave(torch.arange(c["batch"], device="cuda"), lens, output_size=n)
    pos = t["counts"].long()[seq] + torch.arange(n, device="cuda") - t["seq_start"].long()[seq]
    # (angles in 64 bits: at a far position fp32 holds too little of them)
    freq = THETA ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = pos.double()[:, None, None] * freq
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

    out = torch.zeros((n + c["pad"], hq, d), dtype=TORCH[c["out"]], device="cuda")
    out[:n] = turn(q).to(out.dtype)
    at, slot = t["table"].long()[seq, pos // page], pos % page
    t["k_pages"][at, :, slot] = turn(k).to(t["k_pages"].dtype)
    t["v_pages"][at, :, slot] = v.to(t["v_pages"].dtype)
    return out, t["k_pages"], t["v_pages"]


def _plain_attention(c, t):
    new, held = _plan(c)
    starts, hkv, group, d = _starts(new), c["hkv"], c["hq"] // c["hkv"], c["d"]
    out = torch.zeros((starts[-1] + c["pad"], c["hq"], d), dtype=TORCH[c["out"]], device="cuda")
    for s, (n, h) in enumerate(zip(new, held)):
        live = h + n
        pages = t["table"][s, :(live + c["page"] - 1) // c["page"]].long()
        k, v = (t[x][pages].transpose(0, 1).reshape(hkv, -1, d)[:, :live].float() for x in ("k_pages", "v_pages"))
        pos = torch.arange(h, live, device="cuda")[:, None]
        key = torch.arange(live, device="cuda")[None, :]
        see = key <= pos
        if c["span"]:
            see = see & (key > pos - c["span"])
        see = see.repeat_interleave(group, 0)
        q = t["q"][starts[s]:starts[s + 1]].float().view(n, hkv, group, d)
        for i in range(hkv):
            w = q[:, i].reshape(n * group, d) @ k[i].t() / math.sqrt(d)
            w = w.masked_fill(~see, -math.inf)
            e = torch.exp(w - w.amax(-1, keepdim=True))
            o = e @ v[i] / e.sum(-1, keepdim=True)
            out[starts[s]:starts[s + 1], i * group:(i + 1) * group] = o.view(n, group, d).to(out.dtype)
    return out


def _plain_verify(c, t):
    """In 64 bits: a running sum's step past the random number has to fall on the same token."""
    v, batch = c["vocab"], c["batch"]
    index = torch.arange(v, device="cuda")
    last = t["seq_start"][1:].long() - 1
    seq = torch.bucketize(torch.arange(t["target"].shape[0], device="cuda"), last)
    temp = t["temperature"].double()[seq][:, None]

    def probabilities(x):
        x = x.double()
        top = x.amax(-1, keepdim=True)
        lowest = torch.where(x == top, index, v).amin(-1, keepdim=True)
        e = torch.exp((x - top) / torch.where(temp > 0, temp, 1.0))
        return torch.where(temp > 0, e / e.sum(-1, keepdim=True), (index == lowest).double())

    p = probabilities(t["target"])
    token = t["tokens"].long()
    fed = torch.cat((token[1:], token[:1]))[:, None]          # the token that follows a row
    if c["draft"] == "logits":
        q = probabilities(t["draft"])
    else:
        q = (index == fed).double()
    u = t["uniform"].double()
    keep = u * q.gather(1, fed)[:, 0] < p.gather(1, fed)[:, 0]
    row = torch.arange(t["target"].shape[0], device="cuda")
    # the first row of each sequence that is not kept; its last row judges no draft
    stop = torch.where(keep & (row != last[seq]), row.numel(), row)
    at = torch.full((batch,), row.numel(), device="cuda").scatter_reduce_(0, seq, stop, "amin")
    weight = (p[at] - q[at]).clamp_min(0)
    # (a draft that its own distribution rules out can leave nothing)
    weight = torch.where((at == last)[:, None] | (weight.amax(-1, keepdim=True) == 0), p[at], weight)
    run_sum = torch.cumsum(weight, -1)
    past = run_sum > u[last][:, None] * run_sum[:, -1:]
    drawn = torch.where(past, index, v).amin(-1)
    drawn = torch.where(drawn < v, drawn, torch.where(weight > 0, index, 0).amax(-1))
    out = torch.where(row < at[seq], fed[:, 0], -1)
    out[at] = drawn
    accepted = at - t["seq_start"][:-1].long()
    return out.to(torch.int32), accepted.to(torch.int32), (t["counts"] + accepted + 1).to(torch.int32)


# ---- the framework's calls ----------------------------------------------------

class _Dev:
    """A torch tensor as the buffer handle _capi's argument builders take."""

    def __init__(self, t):
        from vai_amd import _capi as capi
        self.t, self.ptr, self.shape = t, t.data_ptr(), tuple(t.shape)
        self.nbytes = t.numel() * t.element_size()
        self.code = {torch.float32: capi.F32, torch.float16: capi.F16}.get(t.dtype)


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
    if c["op"] == "verify":
        rows = t["target"].shape[0]
        out = torch.empty((rows,), dtype=torch.int32, device="cuda")
        accepted, counts = (torch.empty((c["batch"],), dtype=torch.int32, device="cuda") for _ in range(2))
        a = capi.verify_drafts_args(_Dev(out), _Dev(accepted), dev("target"), dev("tokens"), dev("uniform"),
                                    dev("seq_start"), draft=dev("draft"), temperature=dev("temperature"),
                                    counts=dev("counts"), new_counts=_Dev(counts))
        ws = _workspace(a, L.vai_verify_drafts_workspace_size(ctypes.byref(a)))
        return {"call": L.vai_verify_drafts_launch, "args": (ctypes.byref(a), stream), "out": (out, accepted, counts),
                "keep": (a, ws, t)}
    pages = capi.kv_pages(dev("k_pages"), dev("v_pages"), dev("table"), dev("seq_start"), dev("counts"))
    rows = sum(_plan(c)[0]) + c["pad"]
    out = torch.zeros((rows, c["hq"], c["d"]), dtype=TORCH[c["out"]], device="cuda")
    if c["op"] == "append":
        a = capi.paged_append_args(_Dev(out), dev("qkv"), pages, dev("q_weight"), dev("k_weight"), norm=c["norm"],
                                   eps=EPS, theta=THETA, rot_dim=c["rot"], pairs=c["pairs"].upper())
        return {"call": L.vai_paged_append_launch, "args": (ctypes.byref(a), stream),
                "out": (out, t["k_pages"], t["v_pages"]), "keep": (a, t)}
    a = capi.paged_attention_args(_Dev(out), dev("q"), pages, causal=True, span=c["span"],
                                  max_new=max(c["new"], c["chunk"]))
    ws = _workspace(a, L.vai_paged_attention_workspace_size(ctypes.byref(a)))
    return {"call": L.vai_paged_attention_launch, "args": (ctypes.byref(a), stream), "out": out, "keep": (a, ws, t)}


def _own_run(state):
    status = state["call"](*state["args"])
    if status:
        from vai_amd import _capi as capi
        capi.check(status, "launch")
    return state["out"]


# ---- work and 64-bit results ----------------------------------------------------

def work(case):
    c = case
    new, held = _plan(c)
    n = sum(new)
    if c["op"] == "verify":
        v = c["vocab"]
        rows = n + (n - c["batch"] if c["draft"] == "logits" else 0)     # (a last row has no draft to weigh)
        return {"bytes": rows * v * BYTES[c["x"]] + 12 * n + 24 * c["batch"], "flops": 4 * rows * v}
    if c["op"] == "append":
        row, kv = (c["hq"] + 2 * c["hkv"]) * c["d"], 2 * c["hkv"] * c["d"]
        moved = n * (row * BYTES[c["x"]] + c["hq"] * c["d"] * BYTES[c["out"]] + kv * BYTES[c["pages"]])
        return {"bytes": moved + (4 * c["d"] if c["norm"] else 0) + 8 * c["batch"],
                "flops": n * (c["hq"] + c["hkv"]) * c["d"] * (3 + (4 if c["norm"] else 0))}
    pairs = keys = 0
    for a, h in zip(new, held):
        span = c["span"] or h + a
        pairs += sum(min(h + i + 1, span) for i in range(a))
        keys += h + a - max(0, h + 1 - span)
    io = n * c["hq"] * c["d"] * (BYTES[c["x"]] + BYTES[c["out"]])
    return {"bytes": io + 2 * keys * c["hkv"] * c["d"] * BYTES[c["pages"]] + 4 * keys // c["page"],
            "flops": 4 * c["d"] * c["hq"] * pairs}


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    new, held = _plan(c)
    starts = _starts(new)
    if c["op"] == "verify":
        out = torch.full((starts[-1],), -1, dtype=torch.int32)
        accepted, temps = [], t["temperature"].tolist()
        token, u = t["tokens"].tolist(), t["uniform"].double().tolist()

        def spread(name, row, temp):
            x = t[name][row].double()
            if temp == 0:
                best = int((x == x.max()).nonzero()[0, 0])
                return torch.nn.functional.one_hot(torch.tensor(best, device="cuda"), c["vocab"]).double()
            return torch.softmax(x / temp, 0)

        for s, n in enumerate(new):
            a = 0
            while True:
                row = starts[s] + a
                weight = spread("target", row, temps[s])
                if a == n - 1:
                    break
                x = token[row + 1]
                if c["draft"] == "logits":
                    other = spread("draft", row, temps[s])
                else:
                    other = torch.zeros_like(weight)
                    other[x] = 1
                if not u[row] * float(other[x]) < float(weight[x]):
                    rest = torch.relu(weight - other)
                    weight = rest if float(rest.sum()) > 0 else weight
                    break
                out[row] = x
                a += 1
            total = torch.cumsum(weight, 0)
            j = int(torch.searchsorted(total, u[starts[s + 1] - 1] * total[-1], right=True))
            out[row] = min(j, int(weight.nonzero()[-1, 0]))
            accepted.append(a)
        accepted = torch.tensor(accepted, dtype=torch.int32, device="cuda")
        return out.cuda(), accepted, t["counts"] + accepted + 1
    hq, hkv, d, page = c["hq"], c["hkv"], c["d"], c["page"]
    out = torch.zeros((starts[-1] + c["pad"], hq, d), dtype=torch.float64, device="cuda")
    if c["op"] == "append":
        n, half = starts[-1], c["rot"] // 2
        q, k, v = t["qkv"][:n].double().view(n, -1, d).split((hq, hkv, hkv), 1)
        if c["norm"]:
            q = q * (q.square().sum(-1, keepdim=True) / d + EPS).rsqrt() * t["q_weight"].double()
            k = k * (k.square().sum(-1, keepdim=True) / d + EPS).rsqrt() * t["k_weight"].double()
        q, k = q.clone(), k.clone()
        pos = torch.cat([torch.arange(h, h + m, device="cuda") for m, h in zip(new, held)])
        # each pair as a complex number, turned by its angle
        i = torch.arange(half, device="cuda", dtype=torch.float64)
        unit = torch.polar(torch.ones((n, half), dtype=torch.float64, device="cuda"),
                           pos.double()[:, None] * torch.exp(-i * math.log(THETA) / half))[:, None, :]
        lo = torch.arange(half, device="cuda") * (1 if c["pairs"] == "halves" else 2)
        hi = lo + (half if c["pairs"] == "halves" else 1)
        for y in (q, k):
            z = torch.complex(y[..., lo], y[..., hi]) * unit
            y[..., lo], y[..., hi] = z.real, z.imag
        out[:n] = q
        k_pages, v_pages = t["k_pages"].double(), t["v_pages"].double()
        for s, (m, h) in enumerate(zip(new, held)):
            row = starts[s]
            while row < starts[s + 1]:     # page by page
                p = h + row - starts[s]
                take = min(page - p % page, starts[s + 1] - row)
                at = int(t["table"][s, p // page])
                for pages, y in ((k_pages, k), (v_pages, v)):
                    pages[at, :, p % page:p % page + take] = y[row:row + take].transpose(0, 1)
                row += take
        return out, k_pages, v_pages
    group = hq // hkv
    for s, (m, h) in enumerate(zip(new, held)):
        live = h + m
        key = torch.arange(live, device="cuda")
        at = t["table"][s].long()[key // page]
        pos = torch.arange(h, live, device="cuda")[:, None]
        hide = (key > pos) | (key <= pos - c["span"]) if c["span"] else key > pos
        for i in range(hkv):
            k, v = t["k_pages"][at, i, key % page].double(), t["v_pages"][at, i, key % page].double()
            for j in range(i * group, (i + 1) * group):
                w = t["q"][starts[s]:starts[s + 1], j].double() @ k.t() / math.sqrt(d)
                out[starts[s]:starts[s + 1], j] = torch.softmax(w.masked_fill(hide, -math.inf), -1) @ v
    return out

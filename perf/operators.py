"""The prompt path of an inference engine over a paged KV cache, as cases that can be timed.

Four operators: rotary positions on rows of heads (`rope`), rotary positions with the write of
the new keys and values into the pages (`append`), causal attention of packed prompts
(`prompt`), and attention of each sequence's new tokens, one or many, over its paged cache
(`chunk`). `run` takes one pass through one of them, in plain torch or, with `own`, by the C
calls that an engine makes, on a stream of its own with arguments bound once. What an engine
makes once a step for all of its layers (positions, cache slots, the attention's plan) and what
it keeps (frequency table, pages, workspace, output buffers) comes from `prepare`.
"""
import ctypes
import math
import random

import torch

own = False
DEV = "cuda"
_STREAM = []


# ---- the cases ---------------------------------------------------------------------------


def listed():
    return [
        # the query heads of a long prompt's chunk, inside the rows of a fused projection
        {"name": "rope-8192", "op": "rope", "tokens": 8192, "heads": 64, "d": 128, "rot": 128, "layout": "half",
         "scaling": "none", "far": 131072, "x": "bf16", "fused": True, "inverse": False},
        # one token's heads of a model in f32 that rotates pairs side by side in part of the head
        {"name": "rope-1-f32", "op": "rope", "tokens": 1, "heads": 40, "d": 80, "rot": 32, "layout": "interleaved",
         "scaling": "linear", "far": 16000, "x": "f32", "fused": False, "inverse": False},
        # cached keys taken back to position zero, far out in a context stretched by parts
        {"name": "rope-back-1021", "op": "rope", "tokens": 1021, "heads": 8, "d": 256, "rot": 64, "layout": "half",
         "scaling": "yarn", "far": 1000000, "x": "bf16", "fused": False, "inverse": True},
        # a decode step of 64 requests: rotate, and write one row a request into the pages
        {"name": "append-64", "op": "append", "tokens": 64, "heads": 64, "kv_heads": 8, "d": 128, "rot": 128,
         "layout": "half", "scaling": "none", "far": 32768, "x": "bf16", "page": 16},
        # a ragged prefill chunk of the released model's head shape, f32 residual stream
        {"name": "append-2047-f32", "op": "append", "tokens": 2047, "heads": 24, "kv_heads": 2, "d": 256, "rot": 64,
         "layout": "half", "scaling": "yarn", "far": 100000, "x": "f32", "page": 64},
        # one long prompt
        {"name": "prompt-8192", "op": "prompt", "seqs": 1, "longest": 8192, "heads": 32, "kv_heads": 8, "d": 128,
         "q": "bf16", "fused": True},
        # seventeen prompts of different lengths from one token up, packed
        {"name": "prompt-17-ragged", "op": "prompt", "seqs": 17, "longest": 1500, "heads": 64, "kv_heads": 8,
         "d": 128, "q": "bf16", "fused": True},
        # a short prompt, narrow heads, results kept in f32
        {"name": "prompt-333-f32", "op": "prompt", "seqs": 1, "longest": 333, "heads": 16, "kv_heads": 16, "d": 64,
         "q": "f32", "fused": False},
        # the released model's head shape: twelve query heads a KV head, 256 wide
        {"name": "prompt-2048-wide", "op": "prompt", "seqs": 2, "longest": 2048, "heads": 24, "kv_heads": 2, "d": 256,
         "q": "bf16", "fused": False},
        # a prefill chunk of 512 tokens over 16 Ki keys already cached
        {"name": "chunk-512", "op": "chunk", "kind": "chunk", "seqs": 1, "new": 512, "context": 16384, "heads": 64,
         "kv_heads": 8, "d": 128, "page": 16, "q": "bf16"},
        # a decode step of 64 requests, contexts from a few tokens to 8 Ki
        {"name": "chunk-decode-64", "op": "chunk", "kind": "chunk", "seqs": 64, "new": 1, "context": 8191,
         "heads": 64, "kv_heads": 8, "d": 128, "page": 16, "q": "bf16"},
        # one prompt's chunk beside fifteen requests that decode, f32 queries
        {"name": "chunk-mixed-16-f32", "op": "chunk", "kind": "mixed", "seqs": 16, "new": 200, "context": 2500,
         "heads": 32, "kv_heads": 8, "d": 128, "page": 32, "q": "f32"},
    ]


def _log(rng, lo, hi, step=1):
    """An integer spread over the logarithm of [lo, hi], a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, round(v / step) * step)))


def draw(rng):
    op = rng.choice(["rope", "append", "prompt", "prompt", "chunk", "chunk"])
    c = {"op": op}
    if op in ("rope", "append"):
        d = rng.choice([64, 80, 96, 128, 128, 256])
        c.update(tokens=_log(rng, 1, 8192 if op == "rope" else 4096), d=d,
                 rot=rng.choice([d, d, d // 2, d // 4]), layout=rng.choice(["half", "interleaved"]),
                 scaling=rng.choice(["none", "linear", "yarn"]), far=_log(rng, 512, 1000000),
                 x=rng.choice(["bf16", "f32"]))
        if op == "rope":
            c.update(heads=_log(rng, 1, 64 * 128 // max(128, d)), fused=rng.random() < 0.5, inverse=rng.random() < 0.3)
            if c["x"] == "f32":
                c["tokens"] = min(c["tokens"], 4000)
        else:
            hk = rng.choice([1, 2, 4, 8])
            c.update(heads=hk * rng.choice([1, 3, 4, 7, 8]), kv_heads=hk, page=rng.choice([16, 32, 48, 64]))
            if c["heads"] * d > 8192:
                c["tokens"] = min(c["tokens"], 2000)
        return c
    d = rng.choice([64, 128, 128, 256])
    hk = rng.choice([1, 2, 4, 8])
    h = hk * rng.choice([1, 3, 4, 7, 8, 12])
    wide = h * d
    q = rng.choice(["bf16", "bf16", "f32"])
    if op == "prompt":
        seqs = rng.choice([1, 1, 2, 5, 13, 30])
        most = 8192 / math.sqrt(max(1, seqs)) * math.sqrt(4096 / max(4096, 1.1 * wide))
        if q == "f32":
            most *= 0.55
        c.update(seqs=seqs, longest=_log(rng, 1, max(64, int(most * 0.95))), fused=rng.random() < 0.5)
    else:
        kind = rng.choice(["chunk", "chunk", "decode", "decode", "spec", "mixed"])
        seqs = {"chunk": rng.choice([1, 1, 2, 3]), "decode": _log(rng, 1, 128), "spec": _log(rng, 1, 32),
                "mixed": rng.choice([3, 8, 20])}[kind]
        new = {"chunk": _log(rng, 16, 1000), "decode": 1, "spec": rng.randint(2, 8), "mixed": _log(rng, 16, 300)}[kind]
        most = 32768 if kind in ("decode", "spec") else 20000
        cap = min(most, 400_000_000 // (seqs * max(new * h, 4 * hk * d)))
        c.update(kind="mixed" if kind == "mixed" else "chunk", seqs=seqs, new=new,
                 context=_log(rng, new + 1, max(new + 2, cap)), page=rng.choice([16, 32, 48, 64]))
    c.update(heads=h, kv_heads=hk, d=d, q=q)
    return c


def _lens(c):
    """(new tokens, keys) of each sequence, from the case alone: the first is the longest, the
    others spread over the logarithm down to one."""
    rng = random.Random("%s %s %s" % (c["seqs"], c.get("longest", c.get("context")), c.get("new", 0)))
    if c["op"] == "prompt":
        n = [c["longest"]] + [_log(rng, 1, c["longest"]) for _ in range(c["seqs"] - 1)]
        rng.shuffle(n)
        return n, n
    n = [c["new"] if c["kind"] == "chunk" or b == 0 else 1 for b in range(c["seqs"])]
    kv = [c["context"]] + [_log(rng, n[b], c["context"]) for b in range(1, c["seqs"])]
    return n, kv


def _far_scaling(c):
    """The scaling that a case's model has: factor, trained length."""
    return {"none": (1.0, 0), "linear": (4.0, 0), "yarn": (16.0, 8192)}[c["scaling"]]


BASE = 500000.0
BETA_FAST, BETA_SLOW = 32.0, 1.0


def work(c):
    xb = 2 if c.get("x", c.get("q")) == "bf16" else 4
    if c["op"] == "rope":
        n = c["tokens"] * c["heads"] * c["d"]
        return {"bytes": 2 * n * xb + 4 * c["tokens"], "flops": 3 * n}
    if c["op"] == "append":
        nq, nk = c["tokens"] * c["heads"] * c["d"], c["tokens"] * c["kv_heads"] * c["d"]
        return {"bytes": 2 * nq * xb + 2 * nk * (xb + 2) + 12 * c["tokens"], "flops": 3 * (nq + nk)}
    new, kv = _lens(c)
    T, keys = sum(new), sum(kv)
    seen = sum(n * k - n * (n - 1) // 2 for n, k in zip(new, kv))
    return {"bytes": 2 * T * c["heads"] * c["d"] * xb + 2 * 2 * keys * c["kv_heads"] * c["d"],
            "flops": 4 * seen * c["heads"] * c["d"]}


# ---- what an engine has in hand ------------------------------------------------------------


def _dt(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 1000003 + 29) & 0x7FFFFFFF)
    return g


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def _sums(n):
    at = [0]
    for v in n:
        at.append(at[-1] + v)
    return at


def _frequencies(c):
    """Radians a position of each pair, f64, as a model's configuration gives them, and the factor
    on cos and sin."""
    half, (s, trained) = c["rot"] // 2, _far_scaling(c)
    i = torch.arange(half, dtype=torch.float64)
    f = torch.pow(torch.tensor(BASE, dtype=torch.float64), -2.0 * i / c["rot"])
    if c["scaling"] == "linear":
        return (f / s).to(DEV), 1.0
    if c["scaling"] == "yarn":
        turns = lambda b: c["rot"] * math.log(trained / (2 * math.pi * b)) / (2 * math.log(BASE))  # noqa: E731
        lo, hi = max(0, math.floor(turns(BETA_FAST))), min(c["rot"] - 1, math.ceil(turns(BETA_SLOW)))
        r = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return (f * (1.0 - r) + f / s * r).to(DEV), 0.1 * math.log(s) + 1.0
    return f.to(DEV), 1.0


def _inputs(c, seed):
    """The case's tensors, from the seed alone."""
    g = _gen(seed)
    t = {}
    if c["op"] in ("rope", "append"):
        T, H, d = c["tokens"], c["heads"], c["d"]
        dt = _dt(c["x"])
        t["pos"] = torch.randint(0, c["far"], (T,), generator=g, device=DEV, dtype=torch.int32)
        if c["op"] == "rope":
            rows = _randn(g, (T, H + (H // 4 + 1 if c["fused"] else 0), d), dt)
            t["x"] = rows[:, :H]
            return t
        hk, ps = c["kv_heads"], c["page"]
        rows = _randn(g, (T, H + 2 * hk, d), dt)
        t["q"], t["k"], t["v"] = rows[:, :H], rows[:, H:H + hk], rows[:, H + hk:]
        pages = -(-T // ps) + 3
        t["kp"] = _randn(g, (pages, hk, ps, d), torch.bfloat16)
        t["vp"] = _randn(g, (pages, hk, ps, d), torch.bfloat16)
        t["slots"] = torch.randperm(pages * ps, generator=g, device=DEV)[:T].contiguous()
        return t
    new, kv = _lens(c)
    T, H, hk, d = sum(new), c["heads"], c["kv_heads"], c["d"]
    t["cu"] = _ints(_sums(new))
    if c["op"] == "prompt":
        dt = _dt(c["q"])
        if c["fused"] and dt == torch.bfloat16:
            rows = _randn(g, (T, H + 2 * hk, d), dt)
            t["q"], t["k"], t["v"] = rows[:, :H], rows[:, H:H + hk], rows[:, H + hk:]
        else:
            t["q"] = _randn(g, (T, H, d), dt)
            t["k"], t["v"] = (_randn(g, (T, hk, d), torch.bfloat16) for _ in range(2))
        return t
    ps = c["page"]
    t["kv"] = _ints(kv)
    used = [-(-k // ps) for k in kv]
    pages, at = sum(used) + 2, _sums(used)
    perm = torch.randperm(pages, generator=g, device=DEV).int()
    table = torch.zeros((len(kv), max(used)), dtype=torch.int32, device=DEV)
    for b, u in enumerate(used):
        table[b, :u] = perm[at[b]:at[b] + u]
    t["table"] = table
    t["q"] = _randn(g, (T, H, d), _dt(c["q"]))
    t["kp"] = _randn(g, (pages, hk, ps, d), torch.bfloat16)
    t["vp"] = _randn(g, (pages, hk, ps, d), torch.bfloat16)
    return t


def prepare(case, seed):
    c = case
    s = _inputs(c, seed)
    s["case"] = c
    if c["op"] in ("rope", "append"):
        s["freq"], s["mag"] = _frequencies(c)
    else:
        new, kv = _lens(c)
        s["longest"] = (max(new), max(kv))
        s["scale"] = 1.0 / math.sqrt(c["d"])
    if own:
        _engine(s)
    return s


def _stream():
    if not _STREAM:
        _STREAM.append(torch.cuda.Stream())
    return _STREAM[0]


def _engine(s):
    """What an engine keeps (frequency table, workspace, output buffers) and makes once a step (the
    attention's plan), and its call with the arguments bound."""
    import homelab_amd as hip

    c, st = s["case"], _stream()
    torch.cuda.current_stream().synchronize()  # the inputs are written before work on the other stream
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    code = lambda t: hip.BF16 if t.dtype == torch.bfloat16 else hip.F32  # noqa: E731
    stream = ctypes.c_void_p(st.cuda_stream)
    L = hip.lib()
    if c["op"] in ("rope", "append"):
        kind = {"none": hip.ROPE_PLAIN, "linear": hip.ROPE_LINEAR, "yarn": hip.ROPE_YARN}[c["scaling"]]
        layout = {"half": hip.ROPE_HALF, "interleaved": hip.ROPE_INTERLEAVED}[c["layout"]]
        factor, trained = _far_scaling(c)
        turns, mag = hip.rope_table(c["rot"], BASE, kind, factor, trained, BETA_FAST, BETA_SLOW)
        s["turns"] = turns = torch.from_numpy(turns.view("int64")).to(DEV)
        T, H, d = c["tokens"], c["heads"], c["d"]
        if c["op"] == "rope":
            x = s["x"]
            s["out"] = out = torch.empty((T, H, d), dtype=x.dtype, device=DEV)
            args = (p(x), code(x), x.stride(0), p(s["pos"]), p(turns), c["rot"], layout, mag, int(c["inverse"]), p(out),
                    code(out), out.stride(0), T, H, d, stream)
            s["call"], s["outputs"] = (L.oom_rope, args), out
        else:
            q, k, v, kp = s["q"], s["k"], s["v"], s["kp"]
            s["out"] = out = torch.empty((T, H, d), dtype=q.dtype, device=DEV)
            args = (p(q), q.stride(0), p(k), k.stride(0), p(v), v.stride(0), code(q), p(s["pos"]), p(s["slots"]), p(turns),
                    c["rot"], layout, mag, p(out), code(out), out.stride(0), p(kp), p(s["vp"]), kp.shape[0], c["page"], T, H,
                    c["kv_heads"], d, stream)
            s["call"], s["outputs"] = (L.oom_rope_append_paged, args), (out, kp, s["vp"])
    else:
        q, H, hk, d = s["q"], c["heads"], c["kv_heads"], c["d"]
        T, B = q.shape[0], c["seqs"]
        s["out"] = out = torch.empty((T, H, d), dtype=q.dtype, device=DEV)
        s["plan"] = plan = torch.empty(hip.attn_plan_size(T, B, H, hk, d), dtype=torch.int32, device=DEV)
        if c["op"] == "prompt":
            k, v = s["k"], s["v"]
            hip.attn_plan(s["cu"], None, None, T, H, hk, d, plan)
            args = (p(q), code(q), q.stride(0), p(k), k.stride(0), p(v), v.stride(0), p(plan), T, B, H, hk, d, s["scale"],
                    p(out), code(out), out.stride(0), stream)
            s["call"], s["outputs"] = (L.oom_attn_prompt, args), out
        else:
            kp, table = s["kp"], s["table"]
            hip.attn_plan(s["cu"], s["kv"], table, T, H, hk, d, plan, n_pages=kp.shape[0], page_size=c["page"])
            size = hip.attn_chunk_paged_workspace_size(T, B, H, hk, d)
            s["ws"] = ws = torch.zeros(size, dtype=torch.uint8, device=DEV)
            args = (p(q), code(q), q.stride(0), p(kp), p(s["vp"]), p(table), table.shape[1], kp.shape[0], c["page"], p(plan), T,
                    B, s["longest"][0], H, hk, d, s["scale"], p(out), code(out), out.stride(0), p(ws), size, stream)
            s["call"], s["outputs"] = (L.oom_attn_chunk_paged, args), out
    s["check"] = hip.check
    torch.cuda.synchronize()


# ---- one pass --------------------------------------------------------------------------------


def run(state):
    if own:
        fn, args = state["call"]
        state["check"](fn(*args))
        return state["outputs"]
    c = state["case"]
    if c["op"] == "rope":
        x = state["x"]
        return _rotate(x, c, state, -1.0 if c["inverse"] else 1.0).to(x.dtype)
    if c["op"] == "append":
        q = _rotate(state["q"], c, state, 1.0).to(state["q"].dtype)
        k = _rotate(state["k"], c, state, 1.0).to(torch.bfloat16)
        page, at = state["slots"] // c["page"], state["slots"] % c["page"]
        state["kp"][page, :, at] = k
        state["vp"][page, :, at] = state["v"].to(torch.bfloat16)
        return q, state["kp"], state["vp"]
    if c["op"] == "prompt":
        lens = state["cu"].diff().long()
        Lk = state["longest"][1]
        j = torch.arange(Lk, device=DEV)
        row = (state["cu"][:-1].long()[:, None] + j).clamp(max=state["k"].shape[0] - 1)  # [B, keys]
        return _attention(state, lens, lens, state["k"][row], state["v"][row])
    ps, Lk = c["page"], state["longest"][1]
    j = torch.arange(Lk, device=DEV)
    page = state["table"][:, j // ps].long()  # [B, keys]
    return _attention(state, state["cu"].diff().long(), state["kv"].long(), state["kp"][page, :, j % ps],
                      state["vp"][page, :, j % ps])


def _rotate(x, c, state, sign):
    """f32 [T, heads, d]: the first `rot` dims of each head turned by pos f; angles in 64 bits."""
    a = state["pos"].double()[:, None, None] * state["freq"]
    cos, sin = (torch.cos(a) * state["mag"]).float(), (torch.sin(a) * (sign * state["mag"])).float()
    x = x.float()
    r, rest = x[..., :c["rot"]], x[..., c["rot"]:]
    half = c["rot"] // 2
    u, w = (r[..., :half], r[..., half:]) if c["layout"] == "half" else (r[..., 0::2], r[..., 1::2])
    y, z = u * cos - w * sin, u * sin + w * cos
    turned = torch.cat((y, z), -1) if c["layout"] == "half" else torch.stack((y, z), -1).flatten(-2)
    return torch.cat((turned, rest), -1)


def _attention(state, lens, kv, k, v):
    """Each sequence padded to the longest: k and v [B, keys, kv_heads, d], new token i of n at
    position kv - n + i, which sees the keys up to its own."""
    q, (Lq, Lk) = state["q"], state["longest"]
    T, H, d = q.shape
    B, hk = k.shape[0], k.shape[2]
    G = H // hk
    i, j = torch.arange(Lq, device=DEV), torch.arange(Lk, device=DEV)
    first = state["cu"][:-1].long()
    row = (first[:, None] + i).clamp(max=T - 1)
    qf = q[row].float().view(B, Lq, hk, G, d).permute(0, 2, 1, 3, 4).reshape(B, hk, Lq * G, d)
    kf = k.float().permute(0, 2, 3, 1).contiguous()
    vf = v.float().permute(0, 2, 1, 3).contiguous()
    kv, lens = kv[:, None, None], lens[:, None, None]
    sees = (j <= kv - lens + i[:, None]) & (j < kv) & (i[:, None] < lens)  # [B, Lq, Lk]
    s = torch.matmul(qf, kf).view(B, hk, Lq, G, Lk) * state["scale"]
    s = s.masked_fill_(~sees[:, None, :, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min(-3.0e38)
    e = s.sub_(m).exp_()
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(B, hk, Lq * G, Lk), vf).view(B, hk, Lq, G, d)
    o = o / total.clamp_min(1e-38)
    b = torch.repeat_interleave(torch.arange(B, device=DEV), lens.view(-1), output_size=T)
    t = torch.arange(T, device=DEV) - first[b]
    return o[b, :, t].reshape(T, H, d).to(q.dtype)


# ---- the definition in 64 bits -----------------------------------------------------------------


def _turned(x, pos, c, back):
    """Rows [T, heads, d] in 64 bits, one pair of dims at a time."""
    out = x.double().clone()
    half = c["rot"] // 2
    s, trained = _far_scaling(c)
    for i in range(half):
        f = BASE ** (-2.0 * i / c["rot"])
        size = 1.0
        if c["scaling"] == "linear":
            f /= s
        elif c["scaling"] == "yarn":
            at = [c["rot"] * math.log(trained / (2 * math.pi * b)) / (2 * math.log(BASE)) for b in (BETA_FAST, BETA_SLOW)]
            lo, hi = max(0, math.floor(at[0])), min(c["rot"] - 1, math.ceil(at[1]))
            share = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = f * (1.0 - share) + f / s * share
            size = 0.1 * math.log(s) + 1.0
        a = pos.double() * (-f if back else f)
        co, si = (size * torch.cos(a))[:, None], (size * torch.sin(a))[:, None]
        u, w = (i, i + half) if c["layout"] == "half" else (2 * i, 2 * i + 1)
        p, r = x[..., u].double(), x[..., w].double()
        out[..., u] = p * co - r * si
        out[..., w] = p * si + r * co
    return out


def exact(case, seed):
    c = case
    t = _inputs(c, seed)
    if c["op"] == "rope":
        return _turned(t["x"], t["pos"], c, c["inverse"])
    if c["op"] == "append":
        kp, vp = t["kp"].double(), t["vp"].double()
        hk, ps, d = c["kv_heads"], c["page"], c["d"]
        n = kp.shape[0]
        at = ((t["slots"] // ps) * hk * ps + t["slots"] % ps)[:, None] + torch.arange(hk, device=DEV) * ps
        kp.view(n * hk * ps, d)[at.view(-1)] = _turned(t["k"], t["pos"], c, False).reshape(-1, d)
        vp.view(n * hk * ps, d)[at.view(-1)] = t["v"].double().reshape(-1, d)
        return _turned(t["q"], t["pos"], c, False), kp, vp
    new, kv = _lens(c)
    H, hk, d = c["heads"], c["kv_heads"], c["d"]
    out, at = torch.zeros(t["q"].shape, dtype=torch.float64, device=DEV), 0
    for b, (n, keys) in enumerate(zip(new, kv)):
        if c["op"] == "prompt":
            k, v = t["k"][at:at + keys].double(), t["v"][at:at + keys].double()
        else:
            used = t["table"][b, :-(-keys // c["page"])].long()
            k, v = (x[used].double().transpose(1, 2).reshape(-1, hk, d)[:keys] for x in (t["kp"], t["vp"]))
        place = torch.arange(keys - n, keys, device=DEV)
        unseen = torch.arange(keys, device=DEV)[None, :] > place[:, None]
        for h in range(H):
            kh, vh = k[:, h // (H // hk)], v[:, h // (H // hk)]
            for r in range(0, n, 2048):
                s = t["q"][at + r:min(at + r + 2048, at + n), h].double() @ kh.T.contiguous() / math.sqrt(d)
                w = torch.softmax(s.masked_fill(unseen[r:r + 2048], -math.inf), -1)
                out[at + r:at + r + s.shape[0], h] = w @ vh
        at += n
    return out

"""The prompt path's calls together, as an engine makes them: prompts, chunks and decode steps over one
paged cache; in captured graphs, on other streams, at the largest offsets; and what the plan
of a batch holds."""
import math
import random

import pytest
import torch

import prompt_cases as pc

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def hip():
    import homelab_amd

    homelab_amd.lib()  # raises if the library is missing: no fallback
    torch.cuda.init()
    return homelab_amd


class Engine:
    """One layer's attention of a model over a paged cache: what an engine keeps, and a step of it."""

    def __init__(self, hip, H, Hkv, d, rot, page, pages, B, max_pages, dtype, seed=1):
        self.hip, self.H, self.Hkv, self.d, self.page, self.dtype = hip, H, Hkv, d, page, dtype
        self.scale = 1 / math.sqrt(d)
        turns, self.mag = hip.rope_table(rot, 500000.0, hip.ROPE_YARN, 8.0, 4096)
        self.freq = pc.frequencies(rot, 500000.0, "yarn", 8.0, 4096)
        self.turns = torch.from_numpy(turns.view("int64")).cuda()
        self.kp, self.vp = (torch.full((pages, Hkv, page, d), math.nan, dtype=BF, device="cuda") for _ in range(2))
        g = pc.gen(seed)
        self.table = torch.randperm(pages, generator=g, device="cuda")[:B * max_pages].int().view(B, max_pages).contiguous()

    def buffers(self, T):
        hip, B = self.hip, self.table.shape[0]
        size = hip.attn_chunk_paged_workspace_size(T, B, self.H, self.Hkv, self.d)
        return dict(pos=torch.zeros(T, dtype=torch.int32, device="cuda"),
                    slots=torch.zeros(T, dtype=torch.int64, device="cuda"),
                    plan=torch.zeros(hip.attn_plan_size(T, B, self.H, self.Hkv, self.d), dtype=torch.int32, device="cuda"),
                    q=torch.zeros((T, self.H, self.d), dtype=self.dtype, device="cuda"),
                    out=torch.zeros((T, self.H, self.d), dtype=self.dtype, device="cuda"),
                    ws=torch.zeros(size, dtype=torch.uint8, device="cuda"))

    def step(self, rows, cu, kv, max_q, b, stream=None):
        """rows [T, H + 2 Hkv, d]: a fused projection's; kv: keys after the step."""
        hip, H, Hkv = self.hip, self.H, self.Hkv
        T = rows.shape[0]
        hip.attn_plan(cu, kv, self.table, T, H, Hkv, self.d, b["plan"], n_pages=self.kp.shape[0], page_size=self.page,
                      positions=b["pos"], slots=b["slots"], stream=stream)
        hip.rope_append_paged(rows[:, :H], rows[:, H:H + Hkv], rows[:, H + Hkv:], b["pos"], b["slots"], self.turns, b["q"],
                              self.kp, self.vp, hip.ROPE_HALF, self.mag, stream=stream)
        hip.attn_chunk_paged(b["q"], self.kp, self.vp, self.table, b["plan"], max_q, self.scale, b["out"], b["ws"],
                             stream=stream)
        return b["out"]


def turned(e, x, pos):
    return pc.rotate(x, torch.tensor(pos, dtype=torch.int32, device="cuda"), e.freq, 0, e.mag)


@pytest.mark.parametrize("H,Hkv,d,rot,page,dtype", [(8, 2, 128, 128, 16, BF), (12, 1, 256, 64, 32, BF), (6, 3, 64, 64, 48, F32)])
def test_prompt_chunk_and_decode_steps(hip, H, Hkv, d, rot, page, dtype):
    """Three sequences through a prompt step, a ragged chunk step and two decode steps; each step's
    result is attention over everything said so far. The first step also by oom_attn_prompt over
    its own rows, the last also by oom_attn_decode_paged."""
    B, max_pages = 3, 24
    e = Engine(hip, H, Hkv, d, rot, page, B * max_pages + 2, B, max_pages, dtype)
    g = pc.gen(H + d)
    said = [[] for _ in range(B)]  # rows of each sequence
    for new in ([70, 1, 33], [9, 130, 0], [1, 1, 1], [1, 1, 1]):
        T = sum(new)
        rows = pc.randn(g, (T + 2, H + 2 * Hkv, d), dtype)  # two rows of no sequence
        cu, at = pc.cumulative(new), 0
        for b, n in enumerate(new):
            said[b].append(rows[at:at + n].clone())
            at += n
        kv = [sum(x.shape[0] for x in s) for s in said]
        buf = e.buffers(T + 2)
        buf["out"].fill_(5.0)
        kp0 = e.kp.clone()
        e.step(rows, cu, torch.tensor(kv, dtype=torch.int32, device="cuda"), max(new), buf)
        assert buf["pos"][:T].tolist() == [p for b, n in enumerate(new) for p in range(kv[b] - n, kv[b])]
        assert buf["pos"][T:].tolist() == [0, 0] and buf["slots"][T:].tolist() == [-1, -1]
        assert bool((buf["out"][T:] == 5.0).all())
        wrote = (e.kp.view(torch.int16) != kp0.view(torch.int16)).any(-1).any(1).sum()
        assert int(wrote) == T  # the new tokens' slots and no others
        at = 0
        for b, n in enumerate(new):
            if n == 0:
                continue
            # the cache holds bf16 of what the rotation gives: read back, checked, and attended over
            k, v = (pc.unpaged(x, e.table[b], kv[b], page) for x in (e.kp, e.vp))
            every = torch.cat(said[b])
            ks = every[:, H:H + Hkv]
            want_k = turned(e, ks, range(kv[b]))
            p = torch.arange(kv[b], dtype=torch.int32, device="cuda")
            assert bool(((k.double() - want_k).abs() <= pc.rotate_bound(ks, p, e.freq, 0, e.mag, BF)).all())
            assert torch.equal(v, every[:, H + Hkv:].to(BF))
            q = buf["q"][at:at + n]
            bound = pc.rotate_bound(rows[at:at + n, :H], p[kv[b] - n:], e.freq, 0, e.mag, dtype)
            assert bool(((q.double() - turned(e, rows[at:at + n, :H], range(kv[b] - n, kv[b]))).abs() <= bound).all())
            want, tol = pc.attention(q, k, v, e.scale, kv[b] - n, dtype == F32)
            pc.hold(buf["out"][at:at + n], want, tol, f"step {new}, sequence {b}")
            at += n
        if kv == [70, 1, 33]:  # every token of these sequences is in this step
            plan = torch.zeros(hip.attn_plan_size(T, B, H, Hkv, d), dtype=torch.int32, device="cuda")
            hip.attn_plan(cu, None, None, T, H, Hkv, d, plan)
            k, v = (torch.cat([pc.unpaged(x, e.table[b], kv[b], page) for b in range(B)]) for x in (e.kp, e.vp))
            out = torch.empty((T, H, d), dtype=dtype, device="cuda")
            hip.attn_prompt(buf["q"][:T], k, v, plan, B, e.scale, out)
            at = 0
            for b, n in enumerate(new):
                want, tol = pc.attention(buf["q"][at:at + n], k[at:at + n], v[at:at + n], e.scale, 0, dtype == F32)
                pc.hold(out[at:at + n], want, tol, f"prompt, sequence {b}")
                at += n
    if d == 128 and H // Hkv <= 8:
        one = torch.empty((H, d), dtype=F32, device="cuda")
        ws = torch.zeros(hip.attn_decode_workspace_size(kv[1], H, Hkv, d), dtype=torch.uint8, device="cuda")
        hip.attn_decode_paged(buf["q"][1], e.kp, e.vp, e.table[1].contiguous(), kv[1], e.scale, one, ws)
        k, v = (pc.unpaged(x, e.table[1], kv[1], page) for x in (e.kp, e.vp))
        want, tol = pc.attention(buf["q"][1:2], k, v, e.scale, kv[1] - 1, True)
        pc.hold(one[None], want, tol, "decode call")


def test_steps_in_captured_graphs(hip):
    """A decode step and a mixed step captured into two graphs that share a workspace and a cache, replayed
    in turn with new inputs and new lengths, against the same steps made eagerly."""
    H, Hkv, d, page, B, max_pages = 8, 2, 128, 16, 4, 40
    e = Engine(hip, H, Hkv, d, 128, page, B * max_pages, B, max_pages, BF)
    e.kp.normal_(generator=pc.gen(1))
    e.vp.normal_(generator=pc.gen(2))
    kinds = []
    big = e.buffers(B + 60)
    for T, max_q in ((B, 1), (B + 59, 60)):
        b = e.buffers(T)
        b["ws"] = big["ws"]  # one workspace, made for the larger step
        kinds.append(dict(T=T, max_q=max_q, b=b, rows=torch.zeros((T, H + 2 * Hkv, d), dtype=BF, device="cuda"),
                          cu=torch.zeros(B + 1, dtype=torch.int32, device="cuda"),
                          kv=torch.zeros(B, dtype=torch.int32, device="cuda")))
    g, rng = pc.gen(7), random.Random(3)

    def fresh(k):
        k["rows"].copy_(pc.randn(g, tuple(k["rows"].shape), BF))
        n = [1] * B
        n[rng.randrange(B)] += k["T"] - B
        k["cu"].copy_(pc.cumulative(n))
        k["kv"].copy_(torch.tensor([rng.randint(x, max_pages * page) for x in n], dtype=torch.int32, device="cuda"))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for k in kinds:
        fresh(k)
        with torch.cuda.stream(stream):
            e.step(k["rows"], k["cu"], k["kv"], k["max_q"], k["b"])
        stream.synchronize()
        k["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(k["graph"], stream=stream):
            e.step(k["rows"], k["cu"], k["kv"], k["max_q"], k["b"])
    for turn in range(6):
        k = kinds[turn % 2]
        fresh(k)
        torch.cuda.synchronize()
        caches = e.kp.clone(), e.vp.clone()
        k["graph"].replay()
        torch.cuda.synchronize()
        got, after = k["b"]["out"].clone(), (e.kp.clone(), e.vp.clone())
        e.kp.copy_(caches[0])
        e.vp.copy_(caches[1])
        eager = e.buffers(k["T"])
        e.step(k["rows"], k["cu"], k["kv"], k["max_q"], eager)
        torch.cuda.synchronize()
        assert torch.equal(got, eager["out"]), f"replay {turn}"
        assert torch.equal(after[0], e.kp) and torch.equal(after[1], e.vp)


def test_on_another_stream(hip):
    g = pc.gen(15)
    T, H, Hkv, d = 150, 4, 2, 64
    q = pc.randn(g, (T, H, d), BF)
    k, v = (pc.randn(g, (T, Hkv, d), BF) for _ in range(2))
    want, tol = pc.attention(q, k, v, 0.125, 0, False)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    plan = torch.zeros(hip.attn_plan_size(T, 1, H, Hkv, d), dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    hip.attn_plan(pc.cumulative([T]), None, None, T, H, Hkv, d, plan, stream=s)
    hip.attn_prompt(q, k, v, plan, 1, 0.125, out, stream=s)
    s.synchronize()
    pc.hold(out, want, tol)


@pytest.mark.parametrize("d", [64, 256])
def test_two_calls_at_once_share_a_plan(hip, d):
    """Two layers' chunk attention on two streams: one plan, a workspace each; q and out slices of wider rows."""
    g = pc.gen(22 + d)
    H, Hkv, page, new, kv = 8, 2, 16, [90, 1, 3], [2000, 1500, 700]
    T = sum(new)
    plan = torch.zeros(hip.attn_plan_size(T, 3, H, Hkv, d), dtype=torch.int32, device="cuda")
    layers = []
    for i in range(2):
        kp, vp, t = pc.paged(g, kv, Hkv, d, page)
        table = t if i == 0 else layers[0][2]
        if i:  # the second layer's pages lie where the first's do
            kp, vp = (torch.nan_to_num(x) for x in (kp, vp))
        rows = pc.randn(g, (T, H + 3, d), BF)
        ws = torch.full((hip.attn_chunk_paged_workspace_size(T, 3, H, Hkv, d),), 0xFF, dtype=torch.uint8, device="cuda")
        layers.append((kp, vp, table, rows, torch.full((T, H + 2, d), 3.0, dtype=BF, device="cuda"), ws))
    hip.attn_plan(pc.cumulative(new), torch.tensor(kv, dtype=torch.int32, device="cuda"), layers[0][2], T, H, Hkv, d, plan,
                  n_pages=layers[0][0].shape[0], page_size=page)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for _ in range(3):
        for st, (kp, vp, table, rows, out, ws) in zip(streams, layers):
            hip.attn_chunk_paged(rows[:, 2:H + 2], kp, vp, table, plan, max(new), 0.1, out[:, 1:H + 1], ws, stream=st)
    torch.cuda.synchronize()
    for kp, vp, table, rows, out, ws in layers:
        at = 0
        for b, n in enumerate(new):
            k, v = (pc.unpaged(x, table[b], kv[b], page) for x in (kp, vp))
            want, tol = pc.attention(rows[at:at + n, 2:H + 2], k, v, 0.1, kv[b] - n, False)
            pc.hold(out[at:at + n, 1:H + 1], want, tol)
            at += n
        assert bool((out[:, 0] == 3.0).all()) and bool((out[:, H + 1] == 3.0).all())


def test_plan_of_other_sizes_writes_nothing(hip):
    """A plan that was made for another batch, for prompts, or never made leaves the outputs as they were."""
    g = pc.gen(16)
    T, H, Hkv, d, page, kv = 6, 8, 2, 128, 16, [90, 300]
    kp, vp, table = pc.paged(g, kv, Hkv, d, page)
    q = pc.randn(g, (T, H, d), BF)
    size = hip.attn_plan_size(T, 2, H, Hkv, d)
    ws = torch.zeros(hip.attn_chunk_paged_workspace_size(T, 2, H, Hkv, d), dtype=torch.uint8, device="cuda")
    cu, kvt = pc.cumulative([5, 1]), torch.tensor(kv, dtype=torch.int32, device="cuda")
    plans = [torch.zeros(size, dtype=torch.int32, device="cuda"), torch.full((size,), -1, dtype=torch.int32, device="cuda")]
    other = torch.zeros(hip.attn_plan_size(T + 1, 2, H, Hkv, d), dtype=torch.int32, device="cuda")
    hip.attn_plan(cu, kvt, table, T + 1, H, Hkv, d, other, n_pages=kp.shape[0], page_size=page)
    prompt = torch.zeros(size, dtype=torch.int32, device="cuda")
    hip.attn_plan(cu, None, None, T, H, Hkv, d, prompt)
    wide = torch.zeros(size, dtype=torch.int32, device="cuda")
    longer = torch.cat((table, table), 1).contiguous()
    hip.attn_plan(cu, kvt, longer, T, H, Hkv, d, wide, n_pages=kp.shape[0], page_size=page)
    for plan in plans + [other, prompt, wide]:
        for max_q in (1, 5, 40):
            out = torch.full((T, H, d), 3.0, dtype=BF, device="cuda")
            hip.attn_chunk_paged(q, kp, vp, table, plan, max_q, 0.1, out, ws)
            assert bool((out == 3.0).all())
    good = torch.zeros(size, dtype=torch.int32, device="cuda")
    hip.attn_plan(cu, kvt, table, T, H, Hkv, d, good, n_pages=kp.shape[0], page_size=page)
    k, v = (pc.randn(g, (T, Hkv, d), BF) for _ in range(2))
    for plan in plans + [good]:
        out = torch.full((T, H, d), 3.0, dtype=BF, device="cuda")
        hip.attn_prompt(q, k, v, plan, 2, 0.1, out)
        assert bool((out == 3.0).all())


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("T,new,max_q", [(64, [1], 64), (64, [1], 1), (64, [40], 64), (3, [1], 50), (2, [2], 2), (1, [1], 900),
                                         (70, [1, 2], 1000), (70, [60, 0], 64)])
def test_bounds_above_the_lengths(hip, T, new, max_q, d):
    """T and max_q are bounds (of a captured step's buffers): fewer tokens than either are served."""
    g = pc.gen(T + max_q)
    H, Hkv, page = 16, 2, 16
    kv = [300 + n for n in new]
    kp, vp, table = pc.paged(g, kv, Hkv, d, page)
    q = pc.randn(g, (T, H, d), BF)
    B = len(new)
    plan = torch.zeros(hip.attn_plan_size(T, B, H, Hkv, d), dtype=torch.int32, device="cuda")
    hip.attn_plan(pc.cumulative(new), torch.tensor(kv, dtype=torch.int32, device="cuda"), table, T, H, Hkv, d, plan,
                  n_pages=kp.shape[0], page_size=page)
    ws = torch.zeros(hip.attn_chunk_paged_workspace_size(T, B, H, Hkv, d), dtype=torch.uint8, device="cuda")
    out = torch.full((T, H, d), 3.0, dtype=BF, device="cuda")
    hip.attn_chunk_paged(q, kp, vp, table, plan, max(max_q, max(new)), 0.1, out, ws)
    at = 0
    for b, n in enumerate(new):
        k, v = (pc.unpaged(x, table[b], kv[b], page) for x in (kp, vp))
        want, tol = pc.attention(q[at:at + n], k, v, 0.1, kv[b] - n, False)
        pc.hold(out[at:at + n], want, tol)
        at += n
    assert bool((out[at:] == 3.0).all())


def test_lengths_past_the_table_and_sequences_that_share_pages(hip):
    """kv_lens past a sequence's pages are taken as its pages; two sequences may name the same pages."""
    g = pc.gen(17)
    H, Hkv, d, page = 4, 2, 64, 16
    kp, vp, table = pc.paged(g, [64, 64], Hkv, d, page)
    table[1] = table[0]
    q = pc.randn(g, (3, H, d), BF)
    cu = pc.cumulative([2, 1])
    plan = torch.zeros(hip.attn_plan_size(3, 2, H, Hkv, d), dtype=torch.int32, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    kvt = torch.tensor([1 << 30, 63], dtype=torch.int32, device="cuda")
    hip.attn_plan(cu, kvt, table, 3, H, Hkv, d, plan, n_pages=kp.shape[0], page_size=page, positions=pos, slots=slots)
    assert pos.tolist() == [62, 63, 62]
    last = int(table[0, 3]) * page
    assert slots.tolist() == [last + 14, last + 15, last + 14]
    ws = torch.zeros(hip.attn_chunk_paged_workspace_size(3, 2, H, Hkv, d), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    hip.attn_chunk_paged(q, kp, vp, table, plan, 2, 0.125, out, ws)
    k, v = (pc.unpaged(x, table[0], 64, page) for x in (kp, vp))
    for rows, kv in ((slice(0, 2), 64), (slice(2, 3), 63)):
        n = rows.stop - rows.start
        want, tol = pc.attention(q[rows], k[:kv], v[:kv], 0.125, kv - n, False)
        pc.hold(out[rows], want, tol)


def test_batches_that_do_not_rise_touch_nothing_else(hip):
    """cu_q that falls, starts past T or is negative: rows that some sequence claims may hold anything
    finite, no row past the last claim changes and nothing outside is read (its neighbours are NaN)."""
    g = pc.gen(18)
    T, H, Hkv, d = 40, 4, 1, 64
    q = pc.randn(g, (T, H, d), BF)
    k, v = (pc.randn(g, (T, Hkv, d), BF) for _ in range(2))
    for cu in ([0, 30, 10, 20], [-5, 3, 3, 900], [50, 60, 70, 80], [0, 40, 0, 40]):
        cut = torch.tensor(cu, dtype=torch.int32, device="cuda")
        plan = torch.zeros(hip.attn_plan_size(T, 3, H, Hkv, d), dtype=torch.int32, device="cuda")
        hip.attn_plan(cut, None, None, T, H, Hkv, d, plan)
        out = torch.full((T, H, d), 3.0, dtype=BF, device="cuda")
        hip.attn_prompt(q, k, v, plan, 3, 0.125, out)
        assert bool(out.isfinite().all())
        top = max(min(max(c, 0), T) for c in cu)
        if min(cu) >= T:
            assert bool((out == 3.0).all())
        assert bool((out[top:] == 3.0).all())


@pytest.mark.parametrize("cu", [[0, 64, 0, 64], [0, 8, 0, 8, 0, 8, 0], [64, 0, 64, 8, 64, 0], [-70, 64, -1, 90]])
def test_plans_of_overlapping_sequences_hold_nothing_unwritten(hip, cu):
    """Sequences over the same tokens have more rows to merge than the batch has rows: the plan's counts stay
    within what it wrote, and each entry within the batch."""
    g = pc.gen(20)
    T, H, Hkv, d, page, B = 64, 4, 1, 64, 16, len(cu) - 1
    kv = [3000 + b for b in range(B)]
    kp, vp, table = pc.paged(g, kv, Hkv, d, page)
    q = pc.randn(g, (T, H, d), BF)
    plan = torch.full((hip.attn_plan_size(T, B, H, Hkv, d),), -9, dtype=torch.int32, device="cuda")
    hip.attn_plan(torch.tensor(cu, dtype=torch.int32, device="cuda"), torch.tensor(kv, dtype=torch.int32, device="cuda"), table,
                  T, H, Hkv, d, plan, n_pages=kp.shape[0], page_size=page)
    one, two, rows = listed(plan, T, B, H, Hkv, d)
    size = hip.attn_chunk_paged_workspace_size(T, B, H, Hkv, d)
    parts = size // (Hkv * (d + 2) * 4)
    assert one or two
    for q0, r0, r, off, k0, k1, part, b in one + two:
        assert 0 <= b < B and r > 0 and r0 >= 0 and q0 >= 0 and q0 * H + r0 + r <= T * H
        assert 0 <= k0 < k1 <= kv[b] and (part == -1 or 0 <= part <= parts - r)
    for tok, head, part, n in rows:
        assert 0 <= tok < T and 0 <= head < H and part >= 0 and part + (n >> 16) * ((n & 0xffff) - 1) < parts
    out = torch.full((T, H, d), 3.0, dtype=BF, device="cuda")
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    hip.attn_chunk_paged(q, kp, vp, table, plan, T, 0.125, out, ws)
    assert bool(out.isfinite().all())


# ---- the largest offsets ---------------------------------------------------------------------


def test_pages_past_four_gigabytes(hip):
    """Pages whose byte offsets pass 32 bits, read by both chunk kernels and written by the append."""
    g = pc.gen(19)
    H, Hkv, d, page = 16, 8, 128, 64
    n_pages = 36000  # 4.7 GB of K, and of V
    kp, vp = (torch.empty((n_pages, Hkv, page, d), dtype=BF, device="cuda") for _ in range(2))
    used = [35999, 0, 32768, 35001, 17000]
    for p in used:
        kp[p] = pc.randn(g, (Hkv, page, d), BF)
        vp[p] = pc.randn(g, (Hkv, page, d), BF)
    table = torch.tensor([used, used[::-1]], dtype=torch.int32, device="cuda")
    new, kv = [30, 1], [300, 290]
    q = pc.randn(g, (31, H, d), BF)
    cu, kvt = pc.cumulative(new), torch.tensor(kv, dtype=torch.int32, device="cuda")
    plan = torch.zeros(hip.attn_plan_size(31, 2, H, Hkv, d), dtype=torch.int32, device="cuda")
    pos = torch.zeros(31, dtype=torch.int32, device="cuda")
    slots = torch.zeros(31, dtype=torch.int64, device="cuda")
    hip.attn_plan(cu, kvt, table, 31, H, Hkv, d, plan, n_pages=n_pages, page_size=page, positions=pos, slots=slots)
    kn, vn = (pc.randn(g, (31, Hkv, d), BF) for _ in range(2))
    turns, _ = hip.rope_table(d)
    turns = torch.from_numpy(turns.view("int64")).cuda()
    turned_q = torch.empty_like(q)
    hip.rope_append_paged(q, kn, vn, pos, slots, turns, turned_q, kp, vp)
    assert torch.equal(vp[(slots // page), :, slots % page], vn)
    ws = torch.zeros(hip.attn_chunk_paged_workspace_size(31, 2, H, Hkv, d), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    hip.attn_chunk_paged(turned_q, kp, vp, table, plan, 30, 0.09, out, ws)
    for b, rows in enumerate((slice(0, 30), slice(30, 31))):
        k, v = (pc.unpaged(x, table[b], kv[b], page) for x in (kp, vp))
        want, tol = pc.attention(turned_q[rows], k, v, 0.09, kv[b] - new[b], False)
        pc.hold(out[rows], want, tol)


def test_rows_past_two_billion_elements(hip):
    """Token rows whose element offsets pass 31 bits (and more tokens than a grid's second dimension)."""
    g = pc.gen(20)
    T, H, Hkv, d, n = 270000, 64, 8, 128, 66
    x = torch.zeros((T, H, d), dtype=BF, device="cuda")
    x[-n:] = pc.randn(g, (n, H, d), BF)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    turns, _ = hip.rope_table(d)
    turns = torch.from_numpy(turns.view("int64")).cuda()
    y = torch.empty_like(x)
    hip.rope(x, pos, turns, y)
    f = pc.frequencies(d)
    off = (y[-n:].double() - pc.rotate(x[-n:], pos[-n:], f, 0)).abs()
    assert bool((off <= pc.rotate_bound(x[-n:], pos[-n:], f, 0, 1.0, BF)).all())
    assert not bool(y[:1000].any()) and not bool(y[T // 2:T // 2 + 1000].any())
    lens = [n] * (T // n)
    lens[-1] += T - sum(lens)
    assert len(lens) <= 4096
    k, v = (torch.zeros((T, Hkv, d), dtype=BF, device="cuda") for _ in range(2))
    last = lens[-1]
    k[-last:], v[-last:] = pc.randn(g, (last, Hkv, d), BF), pc.randn(g, (last, Hkv, d), BF)
    plan = torch.zeros(hip.attn_plan_size(T, len(lens), H, Hkv, d), dtype=torch.int32, device="cuda")
    hip.attn_plan(pc.cumulative(lens), None, None, T, H, Hkv, d, plan)
    x.fill_(7.0)  # the rotated rows' result goes over their source
    hip.attn_prompt(y, k, v, plan, len(lens), 0.09, x)
    want, tol = pc.attention(y[-last:], k[-last:], v[-last:], 0.09, 0, False)
    pc.hold(x[-last:], want, tol)
    assert not bool(x[:-last].any())  # zero values everywhere else


# ---- the plan -----------------------------------------------------------------------------------


def listed(plan, T, B, H, Hkv, d):
    """(items, few-row items, rows to merge) of a plan as lists of tuples."""
    split, few = -(-(256 if d == 256 else 512) // Hkv), -(-256 // Hkv)
    items, fews = T * (H // Hkv) // 128 + B + split, B + few
    w = plan.tolist()
    n, m, r = w[:3]
    at = 16
    one = [tuple(w[at + 8 * i:at + 8 * i + 8]) for i in range(n)]
    at += 8 * items
    two = [tuple(w[at + 8 * i:at + 8 * i + 8]) for i in range(m)]
    at += 8 * fews
    assert n <= items and m <= fews and at + 4 * r <= len(w)
    return one, two, [tuple(w[at + 4 * i:at + 4 * i + 4]) for i in range(r)]


@pytest.mark.parametrize("seed", range(10))
def test_plan_covers_every_row_and_key_once(hip, seed):
    """Random batches: the items' keys partition what each tile of rows sees, split tiles have partial rows
    of their own, and exactly their rows are listed for the merge."""
    rng = random.Random(seed)
    Hkv = rng.choice([1, 2, 3, 8])
    G = rng.choice([1, 4, 7, 8, 12, 40])
    H, d, page = Hkv * G, rng.choice([64, 128, 256]), 16
    B = rng.choice([1, 3, 40, 600])
    new = [rng.choice([0, 1, 1, 2, rng.randint(1, 400)]) for _ in range(B)]
    kv = [max(0, n + rng.choice([-3, 0, 5, 1000, 20000])) for n in new]
    T = sum(new) + rng.randint(0, 5)
    max_pages = max(1, -(-max(kv) // page))
    table = torch.zeros((B, max_pages), dtype=torch.int32, device="cuda")
    plan = torch.full((hip.attn_plan_size(T, B, H, Hkv, d),), -9, dtype=torch.int32, device="cuda")
    cu = pc.cumulative(new)
    hip.attn_plan(cu, torch.tensor(kv, dtype=torch.int32, device="cuda"), table, T, H, Hkv, d, plan, n_pages=1, page_size=page)
    one, two, rows = listed(plan, T, B, H, Hkv, d)
    few_rows = 16 if d == 256 else 32
    at, tiles = 0, {}
    for b, n in enumerate(new):
        for r0 in range(0, n * G, 128):
            r = min(128, n * G - r0)
            few = n * G <= few_rows and (B > 1 or T * G <= few_rows)
            tiles[(b, r0)] = (at, r, kv[b] - n, max(0, kv[b] - n + (r0 + r - 1) // G + 1), few)
        at += n
    seen, parts, merged = {}, {}, {}
    for few, items in ((False, one), (True, two)):
        for q0, r0, r, off, k0, k1, part, b in items:
            want = tiles[(b, r0)]
            assert (q0, r, off, few) == (want[0], want[1], want[2], want[4])
            assert k0 % 64 == 0
            seen.setdefault((b, r0), []).append((k0, k1, part))
    assert set(seen) == set(tiles)
    for key, spans in seen.items():
        q0, r, off, keys, few = tiles[key]
        spans.sort()
        assert spans[0][0] == 0 and spans[-1][1] == keys
        assert all(a[1] == c[0] for a, c in zip(spans, spans[1:]))
        if len(spans) == 1:
            assert spans[0][2] == -1
            continue
        assert [s[2] for s in spans] == [spans[0][2] + i * r for i in range(len(spans))]
        for x in range(spans[0][2], spans[0][2] + r * len(spans)):
            assert x not in parts
            parts[x] = key
        for i in range(r):
            tok = (key[1] + i) // G
            merged[(q0 + tok, key[1] + i - tok * G)] = (spans[0][2] + i, len(spans) | r << 16, off + tok < 0)
    got = {(e[0], e[1] & 0xffff): (e[2], e[3], bool(e[1] >> 30)) for e in rows}
    assert len(got) == len(rows) and got == merged
    ws_rows = hip.attn_chunk_paged_workspace_size(T, B, H, Hkv, d) // (Hkv * (d + 2) * 4)
    assert not parts or max(parts) < ws_rows


# ---- random batches -----------------------------------------------------------------------------


@pytest.mark.parametrize("seed", range(16))
def test_random_batches(hip, seed):
    rng = random.Random(1000 + seed)
    Hkv, G = rng.choice([1, 2, 3, 4]), rng.choice([1, 2, 5, 8, 12])
    H, d, page = Hkv * G, rng.choice([64, 128, 256]), rng.choice([16, 32, 48, 80])
    B = rng.randint(1, 12)
    new = [rng.choice([0, 1, 1, 3, rng.randint(1, 90)]) for _ in range(B)]
    kv = [max(0, n + rng.choice([-2, 0, 0, 7, 63, 700, 2600])) for n in new]
    qdt, odt = rng.choice([(BF, BF), (BF, BF), (F32, F32), (BF, F32), (F32, BF)])
    print(f"random {new} {kv} H={H} Hkv={Hkv} d={d} page={page} {qdt} {odt}", flush=True)
    g = pc.gen(seed)
    kp, vp, table = pc.paged(g, kv, Hkv, d, page)
    T = sum(new) + 1
    q = pc.randn(g, (T, H, d), qdt)
    # a value that no early token may see, and one that all do
    b = max(range(B), key=lambda i: new[i])
    if kv[b] > 40 and seed % 3 == 0:
        vp[int(table[b, (kv[b] - 1) // page]), 0, (kv[b] - 1) % page, 3] = rng.choice([math.inf, -math.inf, math.nan])
        kp[int(table[b, 0]), Hkv - 1, 1, 0] = rng.choice([-math.inf, math.nan])
    import test_gpu_prompt as tp

    tp.check_chunk(hip, q, kp, vp, table, new, kv, 1 / math.sqrt(d), odt)

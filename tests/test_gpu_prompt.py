"""Causal attention of packed prompts (oom_attn_prompt) and of new tokens over paged caches
(oom_attn_chunk_paged) against 64 bits, through the public wrappers."""
import math

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


def plan_of(hip, lens, H, Hkv, d, T, kv=None, table=None, pages=None):
    cu = pc.cumulative(lens)
    plan = torch.full((hip.attn_plan_size(T, len(lens), H, Hkv, d),), 0x55555555, dtype=torch.int32, device="cuda")
    if kv is None:
        hip.attn_plan(cu, None, None, T, H, Hkv, d, plan)
    else:
        kvt = torch.tensor(kv, dtype=torch.int32, device="cuda")
        hip.attn_plan(cu, kvt, table, T, H, Hkv, d, plan, n_pages=pages.shape[0], page_size=pages.shape[2])
    return plan


def check_prompt(hip, q, k, v, lens, scale, out_dtype, spare=0):
    T, H, d = q.shape
    plan = plan_of(hip, lens, H, k.shape[1], d, T)
    out = torch.full((T, H, d), 7.0, dtype=out_dtype, device="cuda")
    hip.attn_prompt(q, k, v, plan, len(lens), scale, out)
    again = torch.full_like(out, 7.0)
    hip.attn_prompt(q, k, v, plan, len(lens), scale, again)
    assert torch.equal(out.view(torch.uint8), again.view(torch.uint8))  # the same bits
    exact = q.dtype == F32 or out_dtype == F32
    at = 0
    for b, n in enumerate(lens):
        want, tol = pc.attention(q[at:at + n], k[at:at + n], v[at:at + n], scale, 0, exact)
        pc.hold(out[at:at + n], want, tol, f"sequence {b} of {n}")
        at += n
    assert bool((out[at:] == 7.0).all())  # rows behind the last sequence stay as they were
    return out


PROMPTS = [
    # lens, H, Hkv, d, q, out
    ([1], 8, 1, 128, BF, BF),
    ([2, 1, 3], 8, 2, 64, BF, BF),
    ([64], 4, 4, 128, BF, BF),
    ([65, 63, 128, 127, 129], 16, 2, 128, BF, BF),
    ([333, 0, 1, 500, 0], 24, 8, 128, BF, BF),       # empty prompts, three heads a KV head
    ([700], 64, 8, 128, BF, BF),
    ([300, 211], 24, 2, 256, BF, BF),                # twelve heads a KV head
    ([257], 5, 5, 64, BF, BF),
    ([130], 40, 1, 64, BF, F32),                     # forty heads on one KV head
    ([200, 31], 12, 4, 128, F32, F32),
    ([129], 7, 1, 256, F32, BF),
    ([77, 1, 140], 3, 3, 64, F32, F32),
    ([1030], 16, 16, 128, BF, F32),
    ([1500, 17], 9, 3, 64, BF, BF),
]


@pytest.mark.parametrize("lens,H,Hkv,d,qdt,odt", PROMPTS)
def test_prompt(hip, lens, H, Hkv, d, qdt, odt):
    print(f"prompt {lens} H={H} Hkv={Hkv} d={d} {qdt} {odt}", flush=True)
    g = pc.gen(sum(lens) + H)
    T = sum(lens) + 3
    q = pc.randn(g, (T, H, d), qdt)
    k, v = (pc.randn(g, (T, Hkv, d), BF) for _ in range(2))
    check_prompt(hip, q, k, v, lens, 1 / math.sqrt(d), odt)


def test_prompt_slices_of_a_fused_projection(hip):
    """q, k and v as slices of one projection's rows, out as a slice of wider rows."""
    g = pc.gen(5)
    T, H, Hkv, d = 211, 6, 2, 128
    rows = pc.randn(g, (T, H + 2 * Hkv + 1, d), BF)
    q, k, v = rows[:, :H], rows[:, H:H + Hkv], rows[:, H + Hkv:H + 2 * Hkv]
    plan = plan_of(hip, [T], H, Hkv, d, T)
    wide = torch.full((T, H + 2, d), 3.0, dtype=BF, device="cuda")
    hip.attn_prompt(q, k, v, plan, 1, 0.11, wide[:, 1:H + 1])
    want, tol = pc.attention(q, k, v, 0.11, 0, False)
    pc.hold(wide[:, 1:H + 1], want, tol)
    assert bool((wide[:, 0] == 3.0).all()) and bool((wide[:, H + 1] == 3.0).all())


@pytest.mark.parametrize("d,qdt", [(64, BF), (128, BF), (256, BF), (128, F32)])
def test_prompt_ignores_what_later_tokens_hold(hip, d, qdt):
    """NaN and infinities in K and V reach exactly the rows that see their key."""
    g = pc.gen(9 + d)
    T, H, Hkv = 300, 4, 2
    q = pc.randn(g, (T, H, d), qdt)
    k, v = (pc.randn(g, (T, Hkv, d), BF) for _ in range(2))
    v[100, 0, 5] = math.inf
    v[101, 0, d - 1] = -math.inf
    v[150, 1, 17] = math.nan
    v[290, 0, 5] = -math.inf
    k[200, 0, 3] = math.nan
    out = check_prompt(hip, q, k, v, [T], 1 / math.sqrt(d), qdt)
    assert bool(out[:100].isfinite().all()) and bool(out[150:, 2:, 17].isnan().all())
    assert bool(out[200:, :2].isnan().all()) and bool(out[199, 2:, :17].isfinite().all())


@pytest.mark.parametrize("big", [3.0e4, 3.0e38])
def test_prompt_large_scores(hip, big):
    """Scores far past the range of exp: the softmax picks single keys; a key of the lowest
    scores that the type holds weighs nothing beside others, and takes all where it is alone."""
    g = pc.gen(21)
    T, H, d = 190, 2, 64
    q = torch.zeros((T, H, d), dtype=BF, device="cuda")
    q[:, :, 0] = 1.0
    k = torch.zeros((T, 1, d), dtype=BF, device="cuda")
    k[:, 0, 0] = -big
    k[60:, 0, 0] = torch.randint(-100, 100, (T - 60,), generator=g, device="cuda").to(BF)
    v = pc.randn(g, (T, 1, d), BF)
    check_prompt(hip, q, k, v, [T], 1.0, BF)


CHUNKS = [
    # new tokens, keys, H, Hkv, d, page, q, out
    ([1], [1], 8, 1, 128, 16, BF, BF),
    ([1], [4097], 8, 1, 128, 16, BF, BF),                       # one row tile over 17 splits
    ([1] * 9, [1, 2, 16, 17, 63, 64, 65, 700, 1500], 16, 2, 128, 16, BF, BF),
    ([4, 1, 7], [900, 33, 7], 24, 4, 128, 48, BF, BF),          # a page of 48 keys
    ([100], [1300], 64, 8, 128, 16, BF, BF),
    ([130, 1, 1, 0, 1], [130, 77, 300, 50, 0], 8, 2, 128, 64, BF, BF),   # a prompt's first chunk, no tokens, no keys
    ([5, 3], [2, 0], 4, 2, 64, 16, BF, BF),                     # tokens before the first key: rows of zeros
    ([200], [150], 4, 4, 64, 16, BF, BF),                       # fifty rows of zeros
    ([33, 1], [2500, 2500], 24, 2, 256, 32, BF, BF),
    ([1, 1], [777, 3000], 12, 1, 256, 16, F32, F32),
    ([9, 64], [513, 1000], 12, 4, 128, 16, F32, F32),
    ([1, 3, 40], [5000, 64, 129], 5, 5, 64, 32, BF, F32),
    ([2], [9001], 16, 16, 128, 16, F32, BF),
    ([1] * 70, [50 + 13 * i for i in range(70)], 8, 8, 64, 16, BF, BF),
    ([256], [6000], 2, 1, 128, 16, BF, BF),
]


def check_chunk(hip, q, kp, vp, table, new, kv, scale, out_dtype):
    T, H, d = q.shape
    Hkv, page = kp.shape[1], kp.shape[2]
    plan = plan_of(hip, new, H, Hkv, d, T, kv, table, kp)
    size = hip.attn_chunk_paged_workspace_size(T, len(new), H, Hkv, d)
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    out = torch.full((T, H, d), 7.0, dtype=out_dtype, device="cuda")
    hip.attn_chunk_paged(q, kp, vp, table, plan, max(new), scale, out, ws)
    again = torch.full_like(out, 7.0)
    hip.attn_chunk_paged(q, kp, vp, table, plan, max(new), scale, again, ws)
    assert torch.equal(out.view(torch.uint8), again.view(torch.uint8))
    exact = q.dtype == F32 or out_dtype == F32
    at = 0
    for b, n in enumerate(new):
        k, v = (pc.unpaged(x, table[b], kv[b], page) for x in (kp, vp))
        want, tol = pc.attention(q[at:at + n], k, v, scale, kv[b] - n, exact)
        pc.hold(out[at:at + n], want, tol, f"sequence {b}: {n} over {kv[b]}")
        at += n
    assert bool((out[at:] == 7.0).all())
    return out


@pytest.mark.parametrize("new,kv,H,Hkv,d,page,qdt,odt", CHUNKS)
def test_chunk(hip, new, kv, H, Hkv, d, page, qdt, odt):
    print(f"chunk {new} {kv} H={H} Hkv={Hkv} d={d} page={page} {qdt} {odt}", flush=True)
    g = pc.gen(sum(kv) + H)
    T = sum(new) + 2
    kp, vp, table = pc.paged(g, kv, Hkv, d, page)
    q = pc.randn(g, (T, H, d), qdt)
    check_chunk(hip, q, kp, vp, table, new, kv, 1 / math.sqrt(d), odt)


def test_chunk_bad_pages_read_zeros(hip):
    g = pc.gen(31)
    new, kv, H, Hkv, d, page = [20, 1, 1], [300, 600, 90], 8, 2, 128, 16
    kp, vp, table = pc.paged(g, kv, Hkv, d, page)
    table[0, 3], table[0, 18], table[1, 0], table[1, 20], table[2, 5] = -1, kp.shape[0], 1 << 30, -(1 << 31), 1 << 30
    q = pc.randn(g, (sum(new), H, d), BF)
    check_chunk(hip, q, kp, vp, table, new, kv, 0.09, F32)


def test_chunk_values_that_hold_infinities(hip):
    g = pc.gen(32)
    new, kv, H, Hkv, d, page = [70, 1], [200, 500], 4, 2, 128, 16
    kp, vp, table = pc.paged(g, kv, Hkv, d, page)
    vp[int(table[0, 10]), 0, 3, 9] = math.inf    # key 163 of sequence 0: seen from its token 33 on
    vp[int(table[0, 2]), 1, 0, 0] = math.nan     # key 32: seen by all
    vp[int(table[1, 30]), 0, 1, 2] = -math.inf
    q = pc.randn(g, (sum(new), H, d), BF)
    out = check_chunk(hip, q, kp, vp, table, new, kv, 0.09, BF)
    assert bool(out[:33, :2].isfinite().all()) and bool(out[33:70, :2, 9].isinf().all())


def test_chunk_one_token_agrees_with_decode(hip):
    """The one-sequence decode call and the chunk call on the same cache."""
    g = pc.gen(33)
    kv, H, Hkv, d, page = 3000, 32, 8, 128, 16
    kp, vp, table = pc.paged(g, [kv], Hkv, d, page)
    q = pc.randn(g, (1, H, d), BF)
    out = check_chunk(hip, q, kp, vp, table, [1], [kv], 0.088, F32)
    one = torch.empty((H, d), dtype=F32, device="cuda")
    ws = torch.zeros(hip.attn_decode_workspace_size(kv, H, Hkv, d), dtype=torch.uint8, device="cuda")
    hip.attn_decode_paged(q[0], kp, vp, table[0].contiguous(), kv, 0.088, one, ws)
    k, v = (pc.unpaged(x, table[0], kv, page) for x in (kp, vp))
    _, tol = pc.attention(q, k, v, 0.088, kv - 1, True)
    assert bool(((out[0] - one).double().abs() <= 2 * tol[0] + 1e-7).all())


@pytest.mark.parametrize("scale", [0.25, 1.0])
@pytest.mark.parametrize("d,qdt", [(64, BF), (128, BF), (256, BF), (64, F32), (128, F32), (256, F32)])
def test_maxima_that_grow_from_tile_to_tile(hip, d, qdt, scale):
    """Scores that rise along the keys for some rows, fall for others and stay for the rest: the running
    maximum moves in every tile, for a part of a wave's rows; scales on both sides of ln 2."""
    g = pc.gen(41 + d)
    T, H, Hkv, page = 390, 6, 2, 16
    q = 0.1 * pc.randn(g, (T, H, d))
    q[:, :, 0] = torch.randint(-1, 2, (T, H), generator=g, device="cuda").float()
    k, v = (0.1 * pc.randn(g, (T, Hkv, d))).to(BF), pc.randn(g, (T, Hkv, d), BF)
    k[:, :, 0] = (torch.arange(T, device="cuda") // 8 * 4.0).to(BF)[:, None]
    q = q.to(qdt)
    check_prompt(hip, q, k, v, [T - 50, 47], scale, qdt)
    # the same keys in pages: many new tokens (split over the keys), few, one
    kp, vp, table = pc.paged(g, [T] * 3, Hkv, d, page)
    for b in range(3):
        for i in range(0, T, page):
            n = min(page, T - i)
            kp[int(table[b, i // page]), :, :n] = k[i:i + n].transpose(0, 1)
            vp[int(table[b, i // page]), :, :n] = v[i:i + n].transpose(0, 1)
    check_chunk(hip, q[:96], kp, vp, table, [90, 4, 1], [T, T - 3, T], scale, qdt)


@pytest.mark.parametrize("d,qdt", [(128, BF), (256, BF), (128, F32), (256, F32)])
def test_prompt_large_scores_of_wide_heads(hip, d, qdt):
    """test_prompt_large_scores at the other head sizes and fp32 queries."""
    g = pc.gen(43)
    T, H = 190, 2
    q = torch.zeros((T, H, d), dtype=qdt, device="cuda")
    q[:, :, 0] = 1.0
    k = torch.zeros((T, 1, d), dtype=BF, device="cuda")
    k[:, 0, 0] = -3.0e38
    k[60:, 0, 0] = torch.randint(-100, 100, (T - 60,), generator=g, device="cuda").to(BF)
    check_prompt(hip, q, k, pc.randn(g, (T, 1, d), BF), [T], 1.0, qdt)


@pytest.mark.parametrize("d,qdt", [(64, BF), (256, BF), (64, F32), (128, F32), (256, F32)])
def test_chunk_bad_pages_and_infinities_of_every_kernel(hip, d, qdt):
    """Bad pages in the first, a middle and the last tile; infinities and NaN seen by some, all and no rows; of
    a sequence of many rows and of one of few."""
    g = pc.gen(44 + d)
    new, kv, H, Hkv, page = [70, 2], [400, 500], 4, 2, 16
    kp, vp, table = pc.paged(g, kv, Hkv, d, page)
    vp[int(table[0, 23]), 0, 3, 9] = math.inf    # key 371 of sequence 0: seen from its token 41 on
    vp[int(table[0, 2]), 1, 0, d - 1] = math.nan  # key 32: seen by all
    vp[int(table[1, 31]), 0, 3, 2] = -math.inf   # key 499: seen by the last token alone
    kp[int(table[1, 31]), 1, 3, 2] = math.nan
    table[0, 0], table[0, 9], table[0, 24], table[1, 0], table[1, 17] = -1, kp.shape[0], 1 << 30, -(1 << 31), 1 << 30
    q = pc.randn(g, (sum(new), H, d), qdt)
    out = check_chunk(hip, q, kp, vp, table, new, kv, 0.09, qdt)
    assert bool(out[:41, :2].isfinite().all()) and bool(out[41:70, :2, 9].isinf().all())
    assert bool(out[70].isfinite().all()) and bool(out[71, 2:].isnan().all())

"""Rotary positions (oom_rope) and the write of a step's keys and values into the paged cache
(oom_rope_append_paged) against 64 bits, through the public wrappers."""
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


SCALINGS = {
    "plain": dict(base=10000.0),
    "linear": dict(base=500000.0, factor=4.0),
    "yarn": dict(base=500000.0, factor=16.0, trained_len=8192),
    "yarn-short": dict(base=10000.0, factor=3.5, trained_len=300, beta_fast=8.0, beta_slow=2.0),
}


def table(hip, rot, name):
    c = dict(SCALINGS[name])
    kind = {"plain": hip.ROPE_PLAIN, "linear": hip.ROPE_LINEAR}.get(name, hip.ROPE_YARN)
    turns, mag = hip.rope_table(rot, scaling=kind, **c)
    f = pc.frequencies(rot, c["base"], name.split("-")[0], c.get("factor", 1.0), c.get("trained_len", 0),
                       c.get("beta_fast", 32.0), c.get("beta_slow", 1.0))
    want = 0.1 * math.log(c["factor"]) + 1 if name.startswith("yarn") else 1.0
    assert abs(mag - want) <= 2.0 ** -24 * want
    return torch.from_numpy(turns.view("int64")).cuda(), mag, f


def positions(g, T, far):
    p = torch.randint(0, far, (T,), generator=g, device="cuda", dtype=torch.int32)
    p[0] = far - 1
    if T > 2:
        p[1], p[2] = 0, -min(far, 77)
    return p


def within(got, want, bound, what=""):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{what}: worst {float((off - bound).max()):.3g} past its bound"


CASES = [
    # T, heads, d, rot, layout, scaling, far, x, out
    (1, 1, 8, 2, 0, "plain", 10, F32, F32),
    (1, 64, 128, 128, 0, "plain", 32768, BF, BF),
    (70, 8, 128, 128, 1, "plain", 131072, BF, BF),
    (33, 40, 80, 32, 1, "linear", 16000, F32, F32),
    (33, 5, 80, 20, 0, "yarn", 100000, BF, BF),      # half a rotation of 10 dims
    (257, 3, 64, 64, 0, "yarn-short", 1 << 20, F32, BF),
    (19, 24, 256, 64, 0, "yarn", 1 << 30, BF, F32),
    (5, 2, 96, 90, 1, "plain", (1 << 31) - 1, F32, F32),
    (1021, 8, 256, 256, 0, "linear", 5000, BF, BF),
    (3, 7, 1024, 1024, 1, "plain", 5000, F32, F32),
]


@pytest.mark.parametrize("T,H,d,rot,layout,scaling,far,xdt,odt", CASES)
def test_rope(hip, T, H, d, rot, layout, scaling, far, xdt, odt):
    print(f"rope T={T} H={H} d={d} rot={rot} layout={layout} {scaling} far={far} {xdt} {odt}", flush=True)
    g = pc.gen(T + H + rot)
    turns, mag, f = table(hip, rot, scaling)
    pos = positions(g, T, far)
    rows = pc.randn(g, (T, H + 2, d), xdt)
    x = rows[:, 1:H + 1]
    out = torch.full((T, H + 1, d), 9.0, dtype=odt, device="cuda")
    for inverse in (False, True):
        bound = pc.rotate_bound(x, pos, f, layout, mag, odt, inverse)
        hip.rope(x, pos, turns, out[:, :H], layout, mag, inverse)
        within(out[:, :H], pc.rotate(x, pos, f, layout, mag, inverse), bound, f"inverse {inverse}")
        assert torch.equal(out[:, :H, rot:], x[..., rot:].to(odt))
    assert bool((out[:, H] == 9.0).all())
    if xdt == odt:  # in place, inside wider rows
        keep = rows.clone()
        hip.rope(x, pos, turns, x, layout, mag, True)
        assert torch.equal(x, out[:, :H])
        assert torch.equal(rows[:, 0], keep[:, 0]) and torch.equal(rows[:, -1], keep[:, -1])


def test_rope_is_a_rotation(hip):
    """Scores of rotated rows depend on the distance of their positions alone; the inverse undoes it."""
    g = pc.gen(4)
    T, d = 64, 128
    turns, mag, _ = table(hip, d, "plain")
    x = pc.randn(g, (1, 2, d)).expand(T, 2, d).contiguous()
    for start in (0, 1000000):
        pos = (start + 17 * torch.arange(T, device="cuda")).int()
        y = torch.empty_like(x)
        hip.rope(x, pos, turns, y)
        # products of two positions a step apart
        s = (y[1:, 0].double() * y[:-1, 1].double()).sum(-1)
        b = pc.rotate_bound(x, pos, pc.frequencies(d), 0, 1.0, F32).amax() * x.abs().double().sum() * 4
        assert float((s - s[0]).abs().max()) <= float(b)
        z = torch.empty_like(x)
        hip.rope(y, pos, turns, z, inverse=True)
        within(z, x.double(), 3 * pc.rotate_bound(x, pos, pc.frequencies(d), 0, 1.0, F32).amax())


APPENDS = [
    # T, H, Hkv, d, rot, layout, scaling, page, x, q out
    (1, 8, 1, 128, 128, 0, "plain", 16, BF, BF),
    (64, 64, 8, 128, 128, 0, "plain", 16, BF, BF),
    (33, 24, 2, 256, 64, 0, "yarn", 64, F32, F32),
    (200, 6, 3, 80, 32, 1, "linear", 48, BF, F32),
    (17, 4, 4, 64, 10, 0, "plain", 16, F32, BF),
]


@pytest.mark.parametrize("T,H,Hkv,d,rot,layout,scaling,page,xdt,odt", APPENDS)
def test_rope_append(hip, T, H, Hkv, d, rot, layout, scaling, page, xdt, odt):
    print(f"append T={T} H={H} Hkv={Hkv} d={d} rot={rot} {scaling} page={page} {xdt} {odt}", flush=True)
    g = pc.gen(T + d)
    turns, mag, f = table(hip, rot, scaling)
    pos = positions(g, T, 30000)
    rows = pc.randn(g, (T, H + 2 * Hkv, d), xdt)
    q, k, v = rows[:, :H], rows[:, H:H + Hkv], rows[:, H + Hkv:]
    n_pages = -(-T // page) + 2
    kp, vp = (pc.randn(g, (n_pages, Hkv, page, d), BF) for _ in range(2))
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:T].contiguous()
    dropped = torch.zeros(T, dtype=torch.bool, device="cuda")
    if T > 4:
        slots[1], slots[2], slots[3] = -1, n_pages * page, 1 << 40
        dropped[1:4] = True
    k0, v0 = kp.clone(), vp.clone()
    out = torch.empty((T, H, d), dtype=odt, device="cuda")
    hip.rope_append_paged(q, k, v, pos, slots, turns, out, kp, vp, layout, mag)
    within(out, pc.rotate(q, pos, f, layout, mag), pc.rotate_bound(q, pos, f, layout, mag, odt), "q")
    kept = ~dropped
    page_of, at = (slots // page)[kept], (slots % page)[kept]
    within(kp[page_of, :, at], pc.rotate(k, pos, f, layout, mag)[kept],
           pc.rotate_bound(k, pos, f, layout, mag, BF)[kept], "k")
    assert torch.equal(vp[page_of, :, at], v.to(BF)[kept])
    kp[page_of, :, at] = k0[page_of, :, at]
    vp[page_of, :, at] = v0[page_of, :, at]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)  # no other slot was written
    if xdt == odt:  # q in place gives the same bits
        hip.rope_append_paged(q, k, v, pos, slots, turns, q, kp, vp, layout, mag)
        assert torch.equal(q, out)

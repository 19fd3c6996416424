"""Plain 64-bit forms of rotary positions and of attention over packed tokens, the error bounds
that their kernels are held to, and packed and paged inputs (shared by the prompt path's
tests). Everything runs on the device of its inputs."""
import math

import torch


def gen(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=g.device).to(dtype)


def cumulative(lens, device="cuda"):
    return torch.tensor([0] + list(lens), dtype=torch.int32, device=device).cumsum(0, dtype=torch.int32)


# ---- rotary positions ---------------------------------------------------------------------


def frequencies(rot, base=10000.0, scaling="plain", factor=1.0, trained=0, fast=32.0, slow=1.0):
    """f64 radians a position, pair by pair."""
    out = []
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        if scaling == "linear":
            f /= factor
        elif scaling == "yarn":
            dim = lambda beta: rot * math.log(trained / (2 * math.pi * beta)) / (2 * math.log(base))  # noqa: E731
            lo, hi = max(0, math.floor(dim(fast))), min(rot - 1, math.ceil(dim(slow)))
            r = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            f = f * (1 - r) + f / factor * r
        out.append(f)
    return out


def rotate(x, pos, freq, layout, magnitude=1.0, inverse=False):
    """f64 rotation of [T, heads, d] by pos * freq (layout 0: halves, 1: interleaved)."""
    f = torch.tensor(freq, dtype=torch.float64, device=x.device)
    a = pos.double()[:, None, None] * f * (-1.0 if inverse else 1.0)
    c, s = magnitude * torch.cos(a), magnitude * torch.sin(a)
    y, n = x.double().clone(), len(freq)
    i = torch.arange(n, device=x.device)
    u, w = (i, i + n) if layout == 0 else (2 * i, 2 * i + 1)
    p, r = x.double()[..., u], x.double()[..., w]
    y[..., u], y[..., w] = p * c - r * s, p * s + r * c
    return y


def rotate_bound(x, pos, freq, layout, magnitude, dtype, inverse=False):
    """How far the kernel may be off, element by element. The angle: its table entry is f / 2 pi
    rounded to 2^-53 of itself and then to 2^-65 turns (pos times that), the product cut to
    32 bits of a turn and rounded to fp32 (2^-25 of half a turn): 2 pi (2^-32 + |pos| (2^-55 +
    2^-65)) + pi 2^-25 radians in all, twice for the f64 form's own. sin and cos: 2 ulp of
    values up to 1, 2^-22, the factor and two products 2^-23 each. Over |u| + |w|, times the
    magnitude; then half a step of the output type at the result of this direction."""
    a = 2 * (2 * math.pi * (2.0 ** -32 + pos.abs().double() * (2.0 ** -54)) + math.pi * 2.0 ** -25)
    n = len(freq)
    i = torch.arange(n, device=x.device)
    u, w = (i, i + n) if layout == 0 else (2 * i, 2 * i + 1)
    b = torch.zeros_like(x, dtype=torch.float64)
    size = (x.double()[..., u].abs() + x.double()[..., w].abs()) * abs(magnitude)
    e = size * (a[:, None, None] + 2.0 ** -22 + 4 * 2.0 ** -23)
    b[..., u], b[..., w] = e, e
    return b + torch.finfo(dtype).eps / 2 * (rotate(x, pos, freq, layout, magnitude, inverse).abs() + b)


# ---- attention -----------------------------------------------------------------------------


def attention(q, k, v, scale, off, exact):
    """One sequence in 64 bits: q [n, H, d], k and v [keys, Hkv, d], token i at position off + i sees
    the keys up to its own; a token that sees none gets zeros. Returns the result and the
    kernel's error bound, element by element.

    The bound. Scores: d exact products (three bf16 terms of an fp32 q: up to 3 d) summed in fp32,
    |ds| <= 3 (d + 2) 2^-24 A with A the largest scale sum |q k| of a visible pair; the
    exponent's argument rounds twice, 2^-23 of its size (at most 2 A log2 e), the exponential 2^-22: a
    weight's relative error w = (3 (d + 2) + 6) 2^-24 A + 2^-22. Numerator and sum carry it once
    each, their fp32 sums and rescalings another 2 (keys + 64) 2^-24, all over sum p |v|. bf16 on both
    sides: a weight is rounded to bf16 on the way to the numerator, 2^-8 of it. The result then
    rounds to its type, half a step."""
    n, H, d = q.shape
    keys, Hkv = k.shape[0], k.shape[1]
    G = H // Hkv
    out = torch.zeros((n, H, v.shape[2]), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    if keys == 0 or n == 0:
        return out, tol
    pos = off + torch.arange(n, device=q.device)
    seen = torch.arange(keys, device=q.device)[None, :] <= pos[:, None]
    some = seen.any(1)
    qd, kd, vd = q.double(), k.double(), v.double()
    vz = vd.abs().nan_to_num(0.0, 0.0, 0.0)
    for h in range(H):
        kh, vh = kd[:, h // G], vd[:, h // G]
        s = (qd[:, h] @ kh.T.contiguous() * scale).masked_fill(~seen, -math.inf)
        A = float((qd[:, h].abs() @ kh.abs().T.contiguous() * scale).masked_fill(~seen, 0.0).nan_to_num(0.0, 0.0, 0.0).max())
        p = torch.softmax(s, -1)
        # a hidden key has no part, whatever its value holds
        bad = ~vh.isfinite()
        o = p @ torch.where(bad, torch.zeros_like(vh), vh)
        hit = seen.double() @ bad.double() > 0
        if bool(hit.any()):
            pm = p.masked_fill(~seen, 0.0)
            plus = (pm @ (vh == math.inf).double()) > 0
            minus = (pm @ (vh == -math.inf).double()) > 0
            nan = (seen.double() @ vh.isnan().double()) > 0
            o = torch.where(plus, torch.full_like(o, math.inf), o)
            o = torch.where(minus, torch.full_like(o, -math.inf), o)
            o = torch.where(nan | (plus & minus), torch.full_like(o, math.nan), o)
        out[:, h] = torch.where(some[:, None], o, torch.zeros_like(o))
        w = (3 * (d + 2) + 6) * 2.0 ** -24 * A + 2.0 ** -22
        e = (2 * w + 2 * (keys + 64) * 2.0 ** -24 + (0.0 if exact else 2.0 ** -8)) * (p.nan_to_num(0.0) @ vz[:, h // G])
        tol[:, h] = torch.where(some[:, None], e, torch.zeros_like(e))
    return out, tol


def hold(got, want, tol, what=""):
    """Every element of `got` within tol plus half a step of its type; NaN and infinities alike."""
    step = torch.finfo(got.dtype).eps / 2
    g = got.double()
    fine = want.isfinite()
    assert bool((g.isnan() == want.isnan()).all()), f"{what}: NaN in other places"
    assert bool((g[want.isinf()] == want[want.isinf()]).all()), f"{what}: infinities differ"
    lim = tol + step * (want.abs() + tol)
    off = (g - want).abs()
    bad = fine & ~(off <= lim)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} elements outside, worst "
                                 f"{float(((off - lim)[bad]).max()):.3g} over a bound of {float(lim[bad].max()):.3g}")


# ---- packed and paged inputs -----------------------------------------------------------------


def paged(g, kv_lens, Hkv, d, page, spare=2, poison=True):
    """A pool of pages with each sequence's pages in random places: (k_pages, v_pages, table). Slots
    past a sequence's length, and pages of no sequence, hold NaN when poisoned; table entries past
    a sequence's pages name no page."""
    used = [-(-n // page) for n in kv_lens]
    n_pages = sum(used) + spare
    perm = torch.randperm(n_pages, generator=g, device=g.device).int()
    table = torch.full((len(kv_lens), max(used + [1])), -7, dtype=torch.int32, device=g.device)
    kp, vp = (randn(g, (n_pages, Hkv, page, d), torch.bfloat16) for _ in range(2))
    held = torch.zeros((n_pages, page), dtype=torch.bool, device=g.device)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = perm[at:at + u]
        for j in range(u):
            held[int(perm[at + j]), :min(page, kv_lens[b] - j * page)] = True
        at += u
    if poison:
        kp.masked_fill_(~held[:, None, :, None], math.nan)
        vp.masked_fill_(~held[:, None, :, None], math.nan)
    return kp, vp, table


def unpaged(pages, table_row, keys, page):
    """[keys, Hkv, d] of one sequence; a bad page reads zeros."""
    Hkv, d = pages.shape[1], pages.shape[3]
    out = torch.zeros((keys, Hkv, d), dtype=pages.dtype, device=pages.device)
    for j in range(-(-keys // page)):
        p = int(table_row[j])
        if 0 <= p < pages.shape[0]:
            n = min(page, keys - j * page)
            out[j * page:j * page + n] = pages[p, :, :n].transpose(0, 1)
    return out

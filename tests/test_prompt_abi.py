"""The prompt path's entry points on the CPU: the frequency table, sizes, and every refusal of
arguments, before anything touches a device."""
import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

import homelab_amd as hip
import prompt_cases as pc

NULL = ctypes.c_void_p(0)
SOME = ctypes.c_void_p(4096)  # an aligned address that no refused call reads


def refused(rc, text):
    assert rc == hip.ERR_ARG, rc
    assert text in hip.lib().oom_last_error().decode(), hip.lib().oom_last_error()


# ---- the frequency table ---------------------------------------------------------------


@pytest.mark.parametrize("rot,base,scaling,args", [
    (2, 10000.0, "plain", {}), (128, 10000.0, "plain", {}), (64, 500000.0, "linear", {"factor": 4.0}),
    (64, 500000.0, "yarn", {"factor": 16.0, "trained": 8192}), (20, 10000.0, "yarn", {"factor": 3.5, "trained": 300,
                                                                                       "fast": 8.0, "slow": 2.0}),
    (1024, 1e6, "yarn", {"factor": 1.0, "trained": 4096}),
])
def test_rope_table(rot, base, scaling, args):
    kind = {"plain": hip.ROPE_PLAIN, "linear": hip.ROPE_LINEAR, "yarn": hip.ROPE_YARN}[scaling]
    turns, mag = hip.rope_table(rot, base, kind, args.get("factor", 1.0), args.get("trained", 0),
                                args.get("fast", 32.0), args.get("slow", 1.0))
    want = pc.frequencies(rot, base, scaling, **args)
    assert turns.shape == (rot // 2,)
    for t, f in zip(turns.tolist(), want):
        # pow and two divisions of doubles, a few 2^-53 of the value, then a 64-bit fraction
        assert abs(Fraction(t, 1 << 64) - Fraction(f) / Fraction(2 * math.pi)) <= Fraction(f) * Fraction(6, 1 << 53) + Fraction(1, 1 << 64)
    assert mag == np.float32(0.1 * math.log(args["factor"]) + 1.0 if scaling == "yarn" else 1.0)


@pytest.mark.parametrize("kw,text", [
    (dict(rot_dim=3), "rot_dim"), (dict(rot_dim=0), "rot_dim"), (dict(rot_dim=2048), "rot_dim"),
    (dict(rot_dim=64, base=1.0), "base"), (dict(rot_dim=64, base=math.nan), "base"),
    (dict(rot_dim=64, scaling=7), "scaling"), (dict(rot_dim=64, scaling=hip.ROPE_LINEAR, factor=0.5), "factor"),
    (dict(rot_dim=64, scaling=hip.ROPE_YARN, factor=2.0), "trained_len"),
    (dict(rot_dim=64, scaling=hip.ROPE_YARN, factor=2.0, trained_len=100, beta_fast=1.0, beta_slow=2.0), "beta_fast"),
    (dict(rot_dim=64, scaling=hip.ROPE_YARN, factor=math.inf, trained_len=100), "factor"),
])
def test_rope_table_refusals(kw, text):
    with pytest.raises(hip.OomError, match=text):
        hip.rope_table(**kw)


def test_rope_table_null_and_short():
    cfg = hip.Rope(64, 0, 10000.0, 1.0, 0, 32.0, 1.0)
    t, m = np.zeros(32, dtype=np.uint64), ctypes.c_float()
    p = t.ctypes.data_as(ctypes.c_void_p)
    refused(hip.lib().oom_rope_table(NULL, p, 32, ctypes.byref(m)), "null")
    refused(hip.lib().oom_rope_table(ctypes.byref(cfg), NULL, 32, ctypes.byref(m)), "null")
    refused(hip.lib().oom_rope_table(ctypes.byref(cfg), p, 31, ctypes.byref(m)), "smaller")


# ---- rotary calls ------------------------------------------------------------------------


def rope_args(**kw):
    a = dict(x=SOME, xdt=1, xs=1024, pos=SOME, turns=SOME, rot=128, layout=0, mag=1.0, inv=0, out=SOME, odt=1, os=1024,
             T=4, heads=8, d=128)
    a.update(kw)
    return list(a.values()) + [NULL]


@pytest.mark.parametrize("kw,text", [
    (dict(d=12), "head_dim"), (dict(d=1032, xs=8256, os=8256), "head_dim"), (dict(rot=0), "rot_dim"), (dict(rot=7), "rot_dim"),
    (dict(rot=130), "rot_dim"), (dict(layout=2), "layout"), (dict(xdt=3), "x_dtype"), (dict(odt=-1), "out_dtype"),
    (dict(T=-1), "T must"), (dict(heads=0), "heads"), (dict(mag=math.nan), "magnitude"), (dict(xs=1016), "strides"),
    (dict(os=1028), "strides"), (dict(x=NULL), "null"), (dict(pos=NULL), "null"), (dict(turns=NULL), "null"),
    (dict(out=NULL), "null"), (dict(x=ctypes.c_void_p(4104)), "16-byte"), (dict(out=ctypes.c_void_p(4098)), "16-byte"),
])
def test_rope_refusals(kw, text):
    refused(hip.lib().oom_rope(*rope_args(**kw)), text)


def append_args(**kw):
    a = dict(q=SOME, qs=1280, k=SOME, ks=1280, v=SOME, vs=1280, xdt=1, pos=SOME, slots=SOME, turns=SOME, rot=128, layout=0,
             mag=1.0, out=SOME, odt=1, os=1024, kp=SOME, vp=SOME, n_pages=4, page=16, T=4, heads=8, kv_heads=1, d=128)
    a.update(kw)
    return list(a.values()) + [NULL]


@pytest.mark.parametrize("kw,text", [
    (dict(d=12), "head_dim"), (dict(rot=129), "rot_dim"), (dict(kv_heads=0), "kv_heads"), (dict(page=24), "page_size"),
    (dict(n_pages=0), "n_pages"), (dict(ks=120), "strides"), (dict(vs=1281), "strides"), (dict(slots=NULL), "null"),
    (dict(k=NULL), "null"), (dict(vp=NULL), "null"), (dict(kp=ctypes.c_void_p(4104)), "16-byte"),
    (dict(v=ctypes.c_void_p(4100)), "16-byte"),
])
def test_append_refusals(kw, text):
    refused(hip.lib().oom_rope_append_paged(*append_args(**kw)), text)


# ---- attention calls ---------------------------------------------------------------------


def plan_args(**kw):
    a = dict(cu=SOME, kv=SOME, table=SOME, max_pages=4, n_pages=9, page=16, T=5, B=2, heads=8, kv_heads=2, d=128, pos=NULL,
             slots=NULL, plan=SOME)
    a.update(kw)
    return list(a.values()) + [NULL]


@pytest.mark.parametrize("kw,text", [
    (dict(d=96), "head_dim"), (dict(heads=9), "multiple of kv_heads"), (dict(kv_heads=0), "multiple of kv_heads"),
    (dict(B=4097), "4096 sequences"), (dict(T=-1), "sequences"), (dict(T=1 << 29), "2^31 rows"),
    (dict(kv=NULL), "go together"), (dict(table=NULL), "go together"), (dict(page=8), "page_size"),
    (dict(page=40), "page_size"), (dict(n_pages=0), "n_pages"), (dict(max_pages=0), "max_pages"),
    (dict(max_pages=1 << 24), "128 Mi"), (dict(kv=NULL, table=NULL, slots=SOME), "slots"), (dict(plan=NULL), "null"),
    (dict(cu=NULL), "null"), (dict(plan=ctypes.c_void_p(4104)), "16-byte"),
])
def test_plan_refusals(kw, text):
    refused(hip.lib().oom_attn_plan(*plan_args(**kw)), text)


def prompt_args(**kw):
    a = dict(q=SOME, qdt=1, qs=1024, k=SOME, ks=256, v=SOME, vs=256, plan=SOME, T=5, B=2, heads=8, kv_heads=2, d=128, scale=0.1,
             out=SOME, odt=1, os=1024)
    a.update(kw)
    return list(a.values()) + [NULL]


@pytest.mark.parametrize("kw,text", [
    (dict(d=80), "head_dim"), (dict(heads=7), "multiple of kv_heads"), (dict(B=4097), "4096 sequences"),
    (dict(qdt=2), "q_dtype"), (dict(odt=2), "out_dtype"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=1e-30), "scale"), (dict(scale=1e30), "scale"), (dict(qs=1016), "strides"), (dict(ks=248), "strides"),
    (dict(vs=260), "strides"), (dict(os=1030), "strides"), (dict(ks=1 << 25), "strides"), (dict(q=NULL), "null"),
    (dict(k=NULL), "null"), (dict(plan=NULL), "null"), (dict(out=NULL), "null"), (dict(v=ctypes.c_void_p(4104)), "16-byte"),
])
def test_prompt_refusals(kw, text):
    refused(hip.lib().oom_attn_prompt(*prompt_args(**kw)), text)


def chunk_args(**kw):
    a = dict(q=SOME, qdt=1, qs=1024, kp=SOME, vp=SOME, table=SOME, max_pages=4, n_pages=9, page=16, plan=SOME, T=5, B=2, max_q=4,
             heads=8, kv_heads=2, d=128, scale=0.1, out=SOME, odt=1, os=1024, ws=SOME, ws_bytes=1 << 40)
    a.update(kw)
    return list(a.values()) + [NULL]


@pytest.mark.parametrize("kw,text", [
    (dict(d=80), "head_dim"), (dict(heads=7), "multiple of kv_heads"), (dict(T=-2), "sequences"), (dict(max_q=0), "max_q"),
    (dict(page=17), "page_size"), (dict(n_pages=0), "n_pages"), (dict(max_pages=1 << 24), "128 Mi"), (dict(qdt=2), "q_dtype"),
    (dict(odt=5), "out_dtype"), (dict(scale=0.0), "scale"), (dict(qs=1016), "strides"), (dict(os=1020), "strides"),
    (dict(q=NULL), "null"), (dict(table=NULL), "null"), (dict(vp=NULL), "null"), (dict(kp=ctypes.c_void_p(4104)), "16-byte"),
    (dict(ws=ctypes.c_void_p(4096 + 128)), "256-byte"),
])
def test_chunk_refusals(kw, text):
    refused(hip.lib().oom_attn_chunk_paged(*chunk_args(**kw)), text)


def test_chunk_workspace_refusals():
    need = hip.attn_chunk_paged_workspace_size(5, 2, 8, 2, 128)
    for kw in (dict(ws=NULL), dict(ws_bytes=need - 1)):
        assert hip.lib().oom_attn_chunk_paged(*chunk_args(**kw)) == hip.ERR_WORKSPACE
        assert "workspace" in hip.lib().oom_last_error().decode()


def test_nothing_to_do():
    """No tokens: a call returns without a look at its buffers."""
    L = hip.lib()
    none = dict(q=NULL, out=NULL, T=0)
    assert L.oom_attn_prompt(*prompt_args(k=NULL, v=NULL, plan=NULL, **none)) == hip.OK
    assert L.oom_attn_chunk_paged(*chunk_args(kp=NULL, vp=NULL, plan=NULL, table=NULL, ws=NULL, ws_bytes=0, **none)) == hip.OK
    assert L.oom_rope(*rope_args(x=NULL, out=NULL, pos=NULL, T=0)) == hip.OK
    assert L.oom_rope_append_paged(*append_args(k=NULL, slots=NULL, **none)) == hip.OK


def test_sizes_grow_with_the_batch():
    for H, Hkv in ((8, 1), (64, 8), (12, 12), (24, 2)):
        for f in (hip.attn_plan_size, hip.attn_chunk_paged_workspace_size):
            sizes = [[f(T, B, H, Hkv, 128) for T in (1, 2, 7, 64, 1000, 9999)] for B in (1, 2, 70, 4096)]
            assert all(s == sorted(s) for s in sizes) and all(list(c) == sorted(c) for c in zip(*sizes))
            assert sizes[0][0] > 0
    assert hip.attn_plan_size(4, 1, 7, 2, 128) == 0 and hip.attn_chunk_paged_workspace_size(4, 1, 0, 2, 128) == 0


def test_wrappers_refuse_what_they_cannot_pass_on():
    x = torch.zeros((4, 8, 128), dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    turns = torch.zeros(64, dtype=torch.int64)
    with pytest.raises(hip.OomError, match="not on the GPU"):
        hip.rope(x, i, turns, x)
    with pytest.raises(hip.OomError, match="positions"):
        hip.rope(x, i[:3], turns, x)
    with pytest.raises(hip.OomError, match="positions"):
        hip.rope(x, i.long(), turns, x)
    with pytest.raises(hip.OomError, match="contiguous"):
        hip.rope(x.transpose(0, 1), torch.zeros(8, dtype=torch.int32), turns, x)
    with pytest.raises(hip.OomError, match="shape"):
        hip.rope(x, i, turns, x[:, :4])
    k = torch.zeros((4, 2, 128), dtype=torch.bfloat16)
    plan = torch.zeros(hip.attn_plan_size(4, 1, 8, 2, 128), dtype=torch.int32)
    with pytest.raises(hip.OomError, match="bfloat16"):
        hip.attn_prompt(x, k.float(), k.float(), plan, 1, 0.1, x)
    with pytest.raises(hip.OomError, match="plan holds"):
        hip.attn_prompt(x, k, k, plan[:8], 1, 0.1, x)
    with pytest.raises(hip.OomError, match="head_dim"):
        hip.attn_prompt(x, k[..., :64], k[..., :64], plan, 1, 0.1, x)
    pages = torch.zeros((3, 2, 16, 128), dtype=torch.bfloat16)
    table = torch.zeros((1, 3), dtype=torch.int32)
    with pytest.raises(hip.OomError, match="k_pages and v_pages"):
        hip.attn_chunk_paged(x, pages, pages[:2], table, plan, 4, 0.1, x, i)
    with pytest.raises(hip.OomError, match="page_table"):
        hip.attn_plan(torch.zeros(2, dtype=torch.int32), i[:1], table.expand(2, 3), 4, 8, 2, 128, plan)

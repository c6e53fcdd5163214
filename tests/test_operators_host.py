"""Routing, rotary positions and log probabilities without a GPU: refusals before any CUDA call, the frequency table, the row
checks of the callers."""
import ctypes as C
import math
import os

import numpy as np
import pytest

from berth_b200 import Error, _lib, kernels, moe
from berth_b200.kernels import ops
from tests import operator_refs as refs

P = 64  # non-null, never dereferenced: the checks return first


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.SO_PATH):
        _lib.build()
    return _lib.lib()


ROUTE = dict(logits=P, f32=1, ld=64, bias=None, idx=P, w=P, T=2, E=64, k=4, score=0, groups=1, keep=1, gs=0, renorm=1, scale=1.0)


@pytest.mark.parametrize("bad,says", [
    (dict(logits=None), "null"), (dict(idx=None), "null"), (dict(w=None), "null"), (dict(T=0), "positive"), (dict(E=0), "n_experts"),
    (dict(E=1025, ld=1025), "n_experts"), (dict(k=0), "top_k"), (dict(k=33), "top_k"), (dict(E=3, k=4), "top_k"), (dict(ld=63), "row_stride"),
    (dict(score=2), "score"), (dict(groups=0), "n_group"), (dict(groups=33), "n_group"), (dict(groups=5), "n_group"), (dict(keep=0), "topk_group"),
    (dict(groups=4, keep=5), "topk_group"), (dict(groups=32, keep=1), "top_k exceeds"), (dict(groups=4, gs=2), "group_score"),
    (dict(groups=16, E=16, keep=8, gs=1), "at least two"), (dict(scale=float("nan")), "finite"), (dict(f32=2), "logits_fp32")])
def test_route_refusals(lib, bad, says):
    a = {**ROUTE, **bad}
    rc = lib.berth_moe_route(a["logits"], a["f32"], a["ld"], a["bias"], a["idx"], a["w"], a["T"], a["E"], a["k"], a["score"], a["groups"], a["keep"],
                             a["gs"], a["renorm"], a["scale"], None)
    assert rc == -1 and says in moe.last_error() and moe.last_launch() == ""


def test_routed_entry_points_refuse_a_bad_routing(lib):
    bad = _lib.MoeRouting(0, 5, 1, 0, 1, 1.0, None)
    assert lib.berth_moe_router_topk_routed(P, P, None, bad, P, P, P, 1, 128, 64, 4, None) == -1
    assert "n_group" in moe.last_error()
    w = _lib.MoeWeights()
    w.hidden, w.inter, w.n_experts, w.top_k, w.k_bits, w.codebook = 256, 128, 64, 4, 4, 2
    assert lib.berth_moe_layer_routed(C.byref(w), bad, P, 1, P, P, P, P, 1 << 40, None) == -1
    assert "n_group" in moe.last_error()
    assert lib.berth_moe_ep_send_routed(P, 1, P, None, bad, 128, 64, 4, P, P, P, P, P, P, 1 << 40, None) == -1
    assert "n_group" in moe.last_error()
    ptrs = (C.c_void_p * 1)(P)
    assert lib.berth_moe_p2p_send_routed(P, 1, P, None, bad, 128, 64, 4, P, P, P, 0, 1, 1, ptrs, ptrs, ptrs, 8, P, 1 << 40, None) == -1
    assert "n_group" in moe.last_error()


def _rows(**kw):
    a = {**dict(x=P, y=P, norm=None, xt=256, xh=64, yt=256, yh=64, heads=4), **kw}
    return _lib.RopeRows(a["x"], a["y"], a["norm"], a["xt"], a["xh"], a["yt"], a["yh"], a["heads"])


@pytest.mark.parametrize("bad,says", [
    (dict(q=None), "null"), (dict(pos=None), "null"), (dict(f=None), "null"), (dict(q=_rows(x=None)), "q: null"), (dict(k=_rows(y=None)), "k: null"),
    (dict(T=0), "positive"), (dict(dim=513), "head_dim"), (dict(dim=1), "head_dim"), (dict(rot=0), "rot_dim"), (dict(rot=7), "rot_dim"),
    (dict(rot=66), "rot_dim"), (dict(f32=3), "fp32"), (dict(q=_rows(heads=0)), "heads"), (dict(q=_rows(heads=1025)), "heads"),
    (dict(q=_rows(yh=63)), "overlap"), (dict(k=_rows(yt=0)), "overlap"), (dict(q=_rows(xt=512)), "in place"),
    (dict(factor=float("inf")), "finite"), (dict(q=_rows(norm=P), eps=-1.0), "epsilon")])
def test_rope_refusals(lib, bad, says):
    a = {**dict(q=_rows(), k=_rows(), pos=P, f=P, T=3, dim=64, rot=64, inter=0, factor=1.0, eps=1e-6, bias=0.0, f32=0), **bad}
    rc = lib.berth_ops_rope(a["q"], a["k"], a["pos"], a["f"], a["T"], a["dim"], a["rot"], a["inter"], a["factor"], a["eps"], a["bias"], a["f32"], None)
    assert rc == -1 and says in ops.last_error() and ops.last_launch() == ""


LOGPROBS = dict(logits=P, f32=1, ld=100, tokens=P, inv_temp=1.0, lp=P, rank=P, h=P, ti=P, tl=P, n=4, rows=2, vocab=100)


@pytest.mark.parametrize("bad,says", [
    (dict(logits=None), "null"), (dict(ti=None), "null"), (dict(tl=None), "null"), (dict(tokens=None), "null tokens"), (dict(rows=0), "positive"),
    (dict(vocab=0), "positive"), (dict(ld=99), "row_stride"), (dict(n=33), "top_n"), (dict(n=-1), "top_n"), (dict(vocab=3), "top_n"),
    (dict(inv_temp=0.0), "inv_temp"), (dict(inv_temp=-1.0), "inv_temp"), (dict(inv_temp=float("nan")), "inv_temp"), (dict(f32=5), "logits_fp32"),
    (dict(tokens=None, lp=None, rank=None, h=None, n=0), "every output")])
def test_logprobs_refusals(lib, bad, says):
    a = {**LOGPROBS, **bad}
    rc = lib.berth_ops_logprobs(a["logits"], a["f32"], a["ld"], a["tokens"], a["inv_temp"], a["lp"], a["rank"], a["h"], a["ti"], a["tl"], a["n"],
                                a["rows"], a["vocab"], None)
    assert rc == -1 and says in ops.last_error() and ops.last_launch() == ""


def test_callers_refuse_host_tensors(lib):
    torch = pytest.importorskip("torch")
    z = torch.zeros
    with pytest.raises(Error, match="CUDA device"):
        ops.logprobs(z(2, 8), None, None, None, z(2), None, None)
    with pytest.raises(Error, match="CUDA device"):
        ops.rope(z(1, 2, 8), None, z(1, dtype=torch.int32), z(4, dtype=torch.float64), z(1, 2, 8), None)
    with pytest.raises(Error, match="CUDA device"):
        moe.route(z(2, 8), None, z(2, 2, dtype=torch.int32), z(2, 2), 2)


# ------------------------------------------------------------------ frequencies

def _steps(got, want, n):
    assert np.abs(np.array(got) / np.array(want) - 1).max() <= n * 2.0 ** -52


@pytest.mark.parametrize("rot", [2, 4, 26, 64, 128, 512])
@pytest.mark.parametrize("base", [1e4, 1e7])
def test_frequencies_plain_linear_and_scaled_base(rot, base):
    plain = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    f, a = ops.rope_frequencies(rot, base)
    _steps(f, plain, 4)
    assert a == 1.0 and len(f) == rot // 2
    f, a = ops.rope_frequencies(rot, base, "linear", factor=8.0)
    _steps(f, [v / 8 for v in plain], 4)
    assert a == 1.0
    if rot == 2:
        with pytest.raises(Error, match="at least 4"):
            ops.rope_frequencies(rot, base, "ntk", factor=4.0)
    else:
        b = base * 4.0 ** (rot / (rot - 2))
        _steps(ops.rope_frequencies(rot, base, "ntk", factor=4.0)[0], [b ** (-2.0 * i / rot) for i in range(rot // 2)], 64)


def test_frequencies_yarn():
    """The fastest pairs as they were, the slowest divided by the factor, monotone between; the factor on cos and sin."""
    rot, base, ctx, factor = 128, 1e6, 32768, 32.0
    f, a = ops.rope_frequencies(rot, base, "yarn", factor=factor, original_context=ctx)
    plain = np.array([base ** (-2.0 * i / rot) for i in range(rot // 2)])
    turns = ctx * plain / (2 * math.pi)
    ratio = np.array(f) / plain
    assert np.allclose(ratio[turns >= 40], 1.0, rtol=1e-15) and np.allclose(ratio[turns <= 0.8], 1 / factor, rtol=1e-14)
    assert (np.diff(ratio) <= 1e-15).all() and ((ratio < 0.99) & (ratio > 1.01 / factor)).sum() > 5
    assert abs(a - (0.1 * math.log(factor) + 1)) < 1e-7
    lo = math.floor(rot * math.log(ctx / (32 * 2 * math.pi)) / (2 * math.log(base)))
    hi = math.ceil(rot * math.log(ctx / (2 * math.pi)) / (2 * math.log(base)))
    ramp = np.clip((np.arange(rot // 2) - lo) / (hi - lo), 0, 1)
    _steps(f, plain * (1 - ramp) + plain / factor * ramp, 8)
    assert ops.rope_frequencies(rot, base, "yarn", factor=factor, original_context=ctx, attention_factor=1.25)[1] == 1.25


def test_frequencies_llama3():
    rot, base, ctx, factor, low, high = 128, 5e5, 8192, 8.0, 1.0, 4.0
    f, a = ops.rope_frequencies(rot, base, "llama3", factor=factor, original_context=ctx, low_factor=low, high_factor=high)
    want = []
    for i in range(rot // 2):
        v = base ** (-2.0 * i / rot)
        wave = 2 * math.pi / v
        if wave < ctx / high:
            want.append(v)
        elif wave > ctx / low:
            want.append(v / factor)
        else:
            s = (ctx / wave - low) / (high - low)
            want.append((1 - s) * v / factor + s * v)
    _steps(f, want, 16)
    assert a == 1.0


@pytest.mark.parametrize("kw,says", [
    (dict(rot_dim=3), "rot_dim"), (dict(rot_dim=0), "rot_dim"), (dict(rot_dim=514), "rot_dim"), (dict(base=1.0), "base"), (dict(base=float("inf")), "base"),
    (dict(scaling="linear", factor=0.5), "factor"), (dict(scaling="yarn", factor=4.0), "original_context"), (dict(scaling="cubic"), "scaling"),
    (dict(scaling="yarn", factor=4.0, original_context=4096, beta_slow=0.0), "beta"),
    (dict(scaling="llama3", factor=4.0, original_context=4096, low_factor=4.0, high_factor=4.0), "high_factor")])
def test_frequencies_refusals(kw, says):
    with pytest.raises(Error, match=says):
        ops.rope_frequencies(**{**dict(rot_dim=64, base=1e4), **kw})


# ------------------------------------------------------------------ the reference itself, on cases worked out by hand

def test_reference_route_by_hand():
    l = np.array([[0.0, 2.0, 1.0, 2.0]], np.float32)
    idx, w = refs.route(l, None, 2, "softmax", 1, 1, "max", True, 1.0)
    assert idx.tolist() == [[1, 3]] and np.allclose(w, 0.5)
    idx, w = refs.route(l, np.array([3.0, 0, 0, 0], np.float32), 2, "sigmoid", 2, 1, "top2", False, 2.0)
    assert idx.tolist() == [[0, 1]] and np.allclose(w, [[1.0, 2 / (1 + math.exp(-2))]])


def test_reference_logprobs_by_hand():
    got = refs.logprobs(np.array([[0.0, math.log(3.0)]]), np.array([0]), 2, 1.0)
    assert np.allclose(got["logprob"], math.log(0.25)) and got["rank"][0] == 1 and got["top"].tolist() == [[1, 0]]
    assert np.allclose(got["entropy"], -(0.25 * math.log(0.25) + 0.75 * math.log(0.75)))


def test_reference_rope_by_hand():
    x = np.array([[[1.0, 0.0, 5.0]]])
    out, _ = refs.rope(x, np.array([1]), np.array([math.pi / 2]), True, 2.0, None, 0.0, 0.0)
    assert np.allclose(out, [[[0.0, 2.0, 5.0]]])


# ------------------------------------------------------------------ pointers off their elements' boundaries, outputs that overlap

@pytest.mark.parametrize("name", ["logits", "bias", "idx", "w"])
def test_route_refuses_unaligned_pointers(lib, name):
    a = {**ROUTE, name: P + 1 if name == "logits" else P + 2}
    for f32 in (0, 1) if name == "logits" else (1,):
        rc = lib.berth_moe_route(a["logits"], f32, a["ld"], a["bias"], a["idx"], a["w"], a["T"], a["E"], a["k"], a["score"], a["groups"], a["keep"],
                                 a["gs"], a["renorm"], a["scale"], None)
        assert rc == -1 and "not aligned" in moe.last_error()


@pytest.mark.parametrize("bad", [dict(q=_rows(x=P + 1)), dict(q=_rows(y=P + 1)), dict(k=_rows(norm=P + 1)), dict(pos=P + 2), dict(f=P + 4),
                                 dict(q=_rows(x=P + 2), f32=1)])
def test_rope_refuses_unaligned_pointers(lib, bad):
    a = {**dict(q=_rows(), k=_rows(), pos=P, f=P, f32=0), **bad}
    assert lib.berth_ops_rope(a["q"], a["k"], a["pos"], a["f"], 3, 64, 64, 0, 1.0, 1e-6, 0.0, a["f32"], None) == -1
    assert "not aligned" in ops.last_error()


@pytest.mark.parametrize("name,off", [("logits", 2), ("tokens", 2), ("lp", 1), ("rank", 2), ("h", 3), ("ti", 2), ("tl", 2)])
def test_logprobs_refuses_unaligned_pointers(lib, name, off):
    a = {**LOGPROBS, name: P + off}
    rc = lib.berth_ops_logprobs(a["logits"], a["f32"], a["ld"], a["tokens"], a["inv_temp"], a["lp"], a["rank"], a["h"], a["ti"], a["tl"], a["n"],
                                a["rows"], a["vocab"], None)
    assert rc == -1 and "not aligned" in ops.last_error()


@pytest.mark.parametrize("yt,yh", [(64, 64), (128, 64), (255, 64), (-128, 64), (64, 128), (64, 191), (64, -191), (0, 64), (256, 0), (100, 100)])
def test_rope_refuses_outputs_whose_heads_overlap(lib, yt, yh):
    """Three tokens of four heads of 64 (256 or 192 apart is enough): one stride inside what lies along the other."""
    q = _rows(x=2 * P, yt=yt, yh=yh)
    assert lib.berth_ops_rope(q, None, P, P, 3, 64, 64, 0, 1.0, 1e-6, 0.0, 0, None) == -1
    assert "overlap" in ops.last_error()


# ------------------------------------------------------------------ frequencies: ends of the ranges

@pytest.mark.parametrize("ctx,fast,slow", [(1.0, 32.0, 1.0), (4.0, 32.0, 1.0), (6.0, 1.0, 1.0), (100.0, 64.0, 32.0), (100.0, 16.0, 16.0)])
@pytest.mark.parametrize("rot", [2, 64])
def test_yarn_divides_every_pair_of_a_context_too_short_for_any(rot, ctx, fast, slow):
    """ctx / (2 pi) turns of the fastest pair: at most beta_slow, so that every frequency is divided by the factor."""
    assert ctx / (2 * math.pi) < slow
    f, _ = ops.rope_frequencies(rot, 1e4, "yarn", factor=4.0, original_context=ctx, beta_fast=fast, beta_slow=slow)
    _steps(f, [1e4 ** (-2.0 * i / rot) / 4.0 for i in range(rot // 2)], 4)


@pytest.mark.parametrize("ctx,fast,slow", [(1e12, 32.0, 1.0), (2000.0, 2.0, 1e-9), (7.0, 1.0, 1.0), (50.0, 32.0, 1.0)])
def test_yarn_at_the_ends_of_the_pairs(ctx, fast, slow):
    """Bounds outside of the pairs: the formula with both brought into 0 .. rot_dim - 1; a pair of beta_fast turns or more is as it was."""
    rot, base, factor = 64, 1e4, 8.0
    f, _ = ops.rope_frequencies(rot, base, "yarn", factor=factor, original_context=ctx, beta_fast=fast, beta_slow=slow)
    plain = np.array([base ** (-2.0 * i / rot) for i in range(rot // 2)])
    turns = ctx * plain / (2 * math.pi)
    assert (np.array(f)[turns >= fast] == plain[turns >= fast]).all()
    lo = max(math.floor(rot * math.log(ctx / (fast * 2 * math.pi)) / (2 * math.log(base))), 0)
    hi = min(math.ceil(rot * math.log(ctx / (slow * 2 * math.pi)) / (2 * math.log(base))), rot - 1)
    ramp = np.clip((np.arange(rot // 2) - lo) / (hi - lo), 0, 1) if hi > lo else (np.arange(rot // 2) > lo) * 1.0
    _steps(f, plain * (1 - ramp) + plain / factor * ramp, 8)


@pytest.mark.parametrize("rot", [2**32 + 64, -2**32 + 64, 2**31, 10**15, -2, 1 << 40])
def test_frequencies_refuse_a_rot_dim_past_the_c_type(rot):
    """Refused as it is, not as what a C int makes of it, and before a table of that size is asked for."""
    with pytest.raises(Error, match="rot_dim"):
        ops.rope_frequencies(rot, 1e4)


def test_frequencies_refuse_a_scaled_base_past_the_type():
    """base * factor^(rot_dim / (rot_dim - 2)) above the largest double would leave frequencies of zero."""
    with pytest.raises(Error, match="scaled base"):
        ops.rope_frequencies(64, 1e4, "ntk", factor=1e300)
    assert min(ops.rope_frequencies(64, 1e4, "ntk", factor=1e280)[0]) > 0

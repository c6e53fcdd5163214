"""Routing, rotary positions and log probabilities at the ends of what their interfaces allow: far offsets, broadcast inputs, infinite
biases, extreme temperatures, two Python threads."""
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from berth_b200 import moe   # noqa: E402
from berth_b200.kernels import ops   # noqa: E402
from tests import operator_refs as refs   # noqa: E402
from tests.strict import wrong   # noqa: E402


def _room(gb):
    if torch.cuda.get_device_properties(0).total_memory < gb << 30:
        pytest.skip(f"needs {gb} GB")


def _rope_close(got, x, pos, f, interleaved, norm=None):
    want, size = refs.rope(x, pos, f, interleaved, 1.0, norm, 1e-6, 1.0)
    tol = size * (2.0 ** -20 + 17 * 2.0 ** -24) + np.abs(want) * 2.0 ** -11 + 2.0 ** -25
    bad = wrong(got.cpu().double().numpy(), want, tol)
    assert not bad.any(), np.argwhere(bad)[:4]


@pytest.mark.parametrize("along", ["tokens", "heads"])
@pytest.mark.parametrize("rot,interleaved", [(64, False), (64, True), (42, False)])
def test_rope_past_32_bit_offsets(along, rot, interleaved):
    """q read from, and k written to, a buffer in which the last row or head starts past element 2^31."""
    _room(24)
    T, hq, hk, D = 4, 3, 3, 64
    n = (T if along == "tokens" else hq) - 1
    far = (2**31 + 64) // n // 8 * 8 + 8
    strides = (far, D, 1) if along == "tokens" else (D, far, 1)
    src, dst = (torch.empty(n * far + 4 * D, dtype=torch.float16, device="cuda") for _ in range(2))
    r = np.random.default_rng(1)
    x = [torch.from_numpy(r.normal(0, 1, (T, h, D))).half() for h in (hq, hk)]
    q, k_out = src.as_strided((T, hq, D), strides), dst.as_strided((T, hk, D), strides)
    q.copy_(x[0])
    k_out.fill_(float("nan"))
    q_out = torch.full((T, hq, D), float("nan"), dtype=torch.float16, device="cuda")
    pos, f = np.array([7, 1000, 3, 12345], np.int32), np.array([1e4 ** (-2.0 * i / rot) for i in range(rot // 2)])
    norm = torch.from_numpy(r.normal(0, 0.1, D)).bfloat16()
    torch.cuda.synchronize()
    ops.rope(q, x[1].cuda(), torch.from_numpy(pos).cuda(), torch.from_numpy(f).cuda(), q_out, k_out, interleaved, 1.0, norm.cuda(), None, 1e-6, 1.0)
    torch.cuda.synchronize()
    _rope_close(q_out, x[0].numpy(), pos, f, interleaved, norm.double().numpy())
    _rope_close(k_out, x[1].numpy(), pos, f, interleaved)


@pytest.mark.parametrize("rot,interleaved", [(128, False), (128, True), (38, False), (88, False)])
def test_rope_of_broadcast_inputs(rot, interleaved):
    """One head for all, one token for all: inputs of stride zero, outputs of their own."""
    T, H, D = 5, 6, 128
    r = np.random.default_rng(2)
    head = torch.from_numpy(r.normal(0, 1, (T, 1, D))).half()
    token = torch.from_numpy(r.normal(0, 1, (1, H, D))).half()
    pos, f = r.integers(0, 9000, T).astype(np.int32), np.array([1e4 ** (-2.0 * i / rot) for i in range(rot // 2)])
    norm = torch.from_numpy(r.normal(0, 0.1, D)).bfloat16()
    out = [torch.full((T, H, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    ops.rope(head.cuda().expand(T, H, D), token.cuda().expand(T, H, D), torch.from_numpy(pos).cuda(), torch.from_numpy(f).cuda(), *out, interleaved, 1.0,
             norm.cuda(), None, 1e-6, 1.0)
    torch.cuda.synchronize()
    _rope_close(out[0], head.expand(T, H, D).numpy(), pos, f, interleaved, norm.double().numpy())
    _rope_close(out[1], token.expand(T, H, D).numpy(), pos, f, interleaved)


@pytest.mark.parametrize("E", [64, 63])
def test_route_past_32_bit_offsets(E):
    _room(12)
    T, k = 5, 4
    stride = (2**31 + 64) // (T - 1) // 8 * 8 + (8 if E == 64 else 9)
    flat = torch.empty(stride * (T - 1) + E, dtype=torch.float16, device="cuda")
    x = flat.as_strided((T, E), (stride, 1))
    l = np.random.default_rng(3).normal(0, 1, (T, E)).astype(np.float16)
    x.copy_(torch.from_numpy(l))
    idx, w = torch.full((T, k), -7, dtype=torch.int32, device="cuda"), torch.full((T, k), float("nan"), device="cuda")
    torch.cuda.synchronize()
    moe.route(x, None, idx, w, k, score="sigmoid", renormalize=True)
    torch.cuda.synchronize()
    want_idx, want_w = refs.route(l, None, k, "sigmoid", 1, 1, "max", True, 1.0)
    assert (idx.cpu().numpy() == want_idx).all()
    assert not wrong(w.cpu().numpy(), want_w, 80 * 2.0 ** -24 * want_w).any()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep,gs", [(1, 1, "max"), (8, 3, "top2"), (8, 3, "max")])
@pytest.mark.parametrize("E", [64, 256])
def test_infinite_biases(score, groups, keep, gs, E):
    """-inf keeps an expert out as long as others are left, +inf brings it to the front; the weights are those of the scores."""
    T, k = 9, 6
    r = np.random.default_rng(E)
    l = r.normal(0, 1, (T, E)).astype(np.float32)
    l[3, ::5] = -np.inf
    b = r.normal(0, 0.1, E).astype(np.float32)
    few = np.full(E, -np.inf, np.float32)
    few[[1, 9, E - 3]] = 0.5
    for bias in (np.where(np.arange(E) % 3 == 0, -np.inf, b), np.where(np.arange(E) % 17 == 4, np.inf, b), few, np.full(E, -np.inf)):
        bias = bias.astype(np.float32)
        want_idx, want_w = refs.route(l, bias, k, score, groups, keep, gs, False, 1.0)
        idx, w = torch.full((T, k), -7, dtype=torch.int32, device="cuda"), torch.full((T, k), float("nan"), device="cuda")
        moe.route(torch.from_numpy(l).cuda(), torch.from_numpy(bias).cuda(), idx, w, k, score=score, n_group=groups, topk_group=keep, group_score=gs,
                  renormalize=False)
        torch.cuda.synchronize()
        assert (idx.cpu().numpy() == want_idx).all()
        assert not wrong(w.cpu().numpy(), want_w, 80 * 2.0 ** -24 * want_w + 1e-37).any()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep", [(1, 1), (8, 3)])
def test_nan_biases_leave_valid_indices(score, groups, keep):
    T, E, k = 5, 64, 8
    l = np.random.default_rng(4).normal(0, 1, (T, E)).astype(np.float32)
    for bias in (np.full(E, np.nan), np.where(np.arange(E) % 2, np.nan, 0.1)):
        idx, w = torch.full((T, k), -7, dtype=torch.int32, device="cuda"), torch.full((T, k), -1.0, device="cuda")
        moe.route(torch.from_numpy(l).cuda(), torch.from_numpy(bias.astype(np.float32)).cuda(), idx, w, k, score=score, n_group=groups, topk_group=keep)
        torch.cuda.synchronize()
        for row in idx.cpu().numpy():
            assert len(set(row.tolist())) == k and row.min() >= 0 and row.max() < E


@pytest.mark.parametrize("inv_temp", [1e30, 1e18, 1e-18, 1e-30])
@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("R,V", [(5, 3001), (600, 5003)])
def test_logprobs_of_extreme_temperatures(inv_temp, f32, R, V):
    """A distribution on the largest logits alone, or on all of them alike."""
    r = np.random.default_rng(5)
    l = r.normal(0, 3, (R, V))
    l[0, [5, V // 2, V - 1]] = 40.0
    l[1, ::2] = -np.inf
    l[2] = float(np.finfo(np.float32 if f32 else np.float16).min)
    l[3, :] = 0.25
    l = l.astype(np.float32 if f32 else np.float16)
    token = r.integers(0, V, R).astype(np.int32)
    token[:4] = [V // 2, 7, V - 1, 0]
    f, i, n = dict(dtype=torch.float32, device="cuda"), dict(dtype=torch.int32, device="cuda"), 5
    lp, rank, h, top, top_lp = (torch.zeros(R, **f), torch.zeros(R, **i), torch.zeros(R, **f), torch.zeros((R, n), **i), torch.zeros((R, n), **f))
    ops.logprobs(torch.from_numpy(l).cuda(), torch.from_numpy(token).cuda(), lp, rank, h, top, top_lp, None, inv_temp)
    torch.cuda.synchronize()
    want = refs.logprobs(l, token, n, float(np.float32(inv_temp)))
    run = (V / 256 + 64) * 2.0 ** -24
    size = lambda v: np.where(np.isfinite(v), np.abs(v), 0.0)
    assert (rank.cpu().numpy() == want["rank"]).all() and (top.cpu().numpy() == want["top"]).all()
    for got, key in ((lp, "logprob"), (top_lp, "top_logprob")):
        bad = wrong(got.cpu().numpy(), want[key], run + size(want[key]) * 6 * 2.0 ** -24)
        assert not bad.any(), (key, np.argwhere(bad)[:4], want[key][bad][:4], got.cpu().numpy()[bad][:4])
    bad = wrong(h.cpu().numpy(), want["entropy"], 2 * run * (1 + np.abs(want["entropy"])))
    assert not bad.any(), (np.argwhere(bad)[:4], want["entropy"][bad][:4], h.cpu().numpy()[bad][:4])


def test_two_threads_on_streams_of_their_own():
    """Two Python threads launch the three operators at once: the bits of one thread alone, and each thread's own last_launch."""
    r = np.random.default_rng(6)
    T, E, k, D, V = 33, 256, 8, 128, 20011

    def make(seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rn = lambda *s: torch.randn(*s, device="cuda", generator=g)
        return dict(l=rn(T, E), b=rn(E) * 0.02, q=rn(T, 8, D).half(), k=rn(T, 2, D).half(), p=torch.randint(0, 9999, (T,), device="cuda", generator=g).int(),
                    x=rn(T, V) * 3, t=torch.randint(0, V, (T,), device="cuda", generator=g).int())
    inv = torch.tensor([1e4 ** (-2.0 * i / D) for i in range(D // 2)], dtype=torch.float64, device="cuda")

    def outs():
        z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device="cuda")
        return dict(idx=z(T, k, dt=torch.int32), w=z(T, k), q=z(T, 8, D, dt=torch.float16), k=z(T, 2, D, dt=torch.float16), lp=z(T), rank=z(T, dt=torch.int32),
                    h=z(T), top=z(T, 5, dt=torch.int32), top_lp=z(T, 5))

    def step(a, o, stream):
        moe.route(a["l"], a["b"], o["idx"], o["w"], k, score="sigmoid", n_group=8, topk_group=4, group_score="top2", stream=stream)
        ops.rope(a["q"], a["k"], a["p"], inv, o["q"], o["k"], stream=stream)
        ops.logprobs(a["x"], a["t"], o["lp"], o["rank"], o["h"], o["top"], o["top_lp"], stream=stream)
    ins = [make(s) for s in (1, 2)]
    want, got, streams = [outs(), outs()], [outs(), outs()], [torch.cuda.Stream() for _ in ins]
    torch.cuda.synchronize()
    for a, o in zip(ins, want):
        step(a, o, None)
    torch.cuda.synchronize()
    begin, said = threading.Barrier(2), [None, None]

    def work(i):
        try:
            begin.wait(30)
            for _ in range(200):
                step(ins[i], got[i], streams[i])
            said[i] = ops.last_launch()
        except Exception as e:   # (looked at below)
            said[i] = e
    ts = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    assert all(isinstance(s, str) and s.startswith("k_logprobs") for s in said), said
    for a, b in zip(want, got):
        assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("V", [40, 3001, 100003])
def test_log_probabilities_of_certain_rows(V, f32):
    """Rows whose largest logit holds all but 10^-4 to 10^-16: ln p and entropy are small numbers, off by at most the roundings at the
    maximum's 1 in its own step (five levels of a tree, half a step of 2^-23 each) and by their own relative errors."""
    r = np.random.default_rng(V)
    gaps = np.array([9.0, 12.0, 15.0, 17.0, 19.0, 23.0, 30.0])
    at = np.array([0, 7, V // 3, V // 2, V - 2, V - 1, 11])
    l = -(np.log(V) + gaps[:, None] + r.uniform(0, 2, (len(gaps), V)))
    l[np.arange(len(gaps)), at] = 0.0
    l = l.astype(np.float32 if f32 else np.float16)
    f, i = dict(dtype=torch.float32, device="cuda"), dict(dtype=torch.int32, device="cuda")
    R = len(gaps)
    lp, rank, h = torch.full((R,), float("nan"), **f), torch.full((R,), -7, **i), torch.full((R,), float("nan"), **f)
    torch.cuda.synchronize()
    ops.logprobs(torch.from_numpy(l).cuda(), torch.from_numpy(at.astype(np.int32)).cuda(), lp, rank, h, None, None)
    torch.cuda.synchronize()
    x = l.astype(np.float64)
    rest = np.where(x == 0, 0.0, np.exp(x)).sum(1)          # z - 1, without the 1
    want_lp = -np.log1p(rest)
    want_h = -want_lp - np.where(x == 0, 0.0, np.exp(x) * x).sum(1) / (1 + rest)
    assert (rank.cpu().numpy() == 0).all()
    # relative: an exponent of up to 62 binary orders, 2.8 units of 2^-24 each, 2^y 4, sums and joins (no more than V / 512 steps) 36
    rel = (2.8 * 62 + 4 + 36 + 3 * (V // 512 + 1)) * 2.0 ** -24
    for got, want in ((lp, want_lp), (h, want_h)):
        bad = wrong(got.cpu().numpy(), want, 5 * 2.0 ** -24 + 2 * rel * np.abs(want))
        assert not bad.any(), (np.argwhere(bad).ravel(), want[bad], got.cpu().numpy()[bad])

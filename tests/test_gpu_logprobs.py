"""Log probabilities, entropy, ranks and alternatives against the definition in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from berth_b200 import Error, kernels   # noqa: E402
from berth_b200.kernels import ops   # noqa: E402
from tests import operator_refs as refs   # noqa: E402


def _call(l, tokens, top, inv_temp=1.0, pad=0, shift=0, stream=None):
    """l numpy [R][V]; rows padded by NaN columns, the first row `shift` elements into its buffer."""
    R, V = l.shape
    dt = torch.float32 if l.dtype == np.float32 else torch.float16
    flat = torch.full((shift + R * (V + pad),), float("nan"), dtype=dt, device="cuda")
    x = flat[shift:].view(R, V + pad)
    x[:, :V] = torch.from_numpy(l).cuda()
    f32, i32 = dict(dtype=torch.float32, device="cuda"), dict(dtype=torch.int32, device="cuda")
    o = {"logprob": torch.full((R + 1,), -7.0, **f32), "rank": torch.full((R + 1,), -7, **i32), "entropy": torch.full((R + 1,), -7.0, **f32),
         "top": torch.full((R + 1, top), -7, **i32), "top_logprob": torch.full((R + 1, top), -7.0, **f32)}
    t = None if tokens is None else torch.from_numpy(np.asarray(tokens, np.int32)).cuda()
    torch.cuda.synchronize()
    ops.logprobs(x, t, o["logprob"][:R] if t is not None else None, o["rank"][:R] if t is not None else None, o["entropy"][:R], o["top"][:R],
                 o["top_logprob"][:R], V, inv_temp, stream=stream)
    torch.cuda.synchronize()
    for v in o.values():
        assert (v[R] == -7).all()                # the row behind the last is left as it was
    return {k: v[:R].cpu().numpy() for k, v in o.items()}


def _check(l, tokens, top, inv_temp=1.0, **kw):
    got = _call(l, tokens, top, inv_temp, **kw)
    want = refs.logprobs(l, tokens, top, inv_temp)
    V = l.shape[1]
    # exponent y = (x - max) * inv_temp * log2 e: two roundings of its factor and one of the product, half a step each; 2^y two
    # steps; a sum of V terms: at most V / 256 of them one after the other, then some 40 joins; log2 and the last product a step each
    run = (V / 256 + 64) * 2.0 ** -24
    def near(a, b, tol, what):
        assert (np.isnan(a) == np.isnan(b)).all(), what
        inf = np.isinf(b)
        assert (a[inf] == b[inf]).all(), what
        ok = np.isnan(b) | inf | (np.abs(a - np.where(inf, 0, b)) <= tol)
        assert ok.all(), (what, a[~ok][:3], b[~ok][:3])
    near(got["entropy"], want["entropy"], 2 * run * (1 + np.abs(want["entropy"])), "entropy")
    near(got["top_logprob"], want["top_logprob"], run + np.abs(want["top_logprob"]) * 6 * 2.0 ** -24, "top_logprob")
    assert (got["top"] == want["top"]).all()
    if tokens is not None:
        near(got["logprob"], want["logprob"], run + np.abs(want["logprob"]) * 6 * 2.0 ** -24, "logprob")
        assert (got["rank"] == want["rank"]).all(), (got["rank"], want["rank"])
    return got


def _rows(seed, R, V, f32, masked=0.0):
    r = np.random.default_rng(seed)
    l = r.normal(0, 2.5, (R, V))
    likely = r.integers(0, V, (R, 4))
    np.put_along_axis(l, likely, r.uniform(0, 18, (R, 4)), 1)
    if masked:
        l[r.random((R, V)) < masked] = -np.inf
        l[:, V // 2] = 1.5
    return l.astype(np.float32 if f32 else np.float16), np.where(r.random(R) < 0.5, likely[:, 0], r.integers(0, V, R)).astype(np.int32)


VOCABS = [1, 2, 7, 31, 33, 255, 1000, 4097, 32003, 100003, 248320]


@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("f32", [True, False])
@pytest.mark.parametrize("masked", [0.0, 0.6])
def test_logprobs_against_the_definition(V, f32, masked):
    for R, top, inv_temp, pad, shift in ((1, 20, 1.25, 0, 0), (3, 32, 1.0, 5, 1), (2, 5, 0.7, 3, 3), (2, 0, 1.0, 1, 0), (1, 1, 1.0, 0, 2)):
        l, tokens = _rows(V + R, R, V, f32, masked)
        _check(l, tokens, min(top, V), inv_temp, pad=pad, shift=shift)


@pytest.mark.parametrize("R,V,f32", [(17, 8192, True), (70, 5003, False), (150, 3001, True), (300, 1030, False), (600, 300, True)])
def test_logprobs_many_rows(R, V, f32):
    """Row counts that leave a block several rows' neighbours: every split of a row over blocks."""
    l, tokens = _rows(R, R, V, f32, 0.1)
    _check(l, tokens, 7, pad=V % 3)


@pytest.mark.parametrize("V", [40, 3000, 70001])
@pytest.mark.parametrize("f32", [True, False])
def test_logprobs_masked_infinite_and_equal_rows(V, f32):
    dt = np.float32 if f32 else np.float16
    low = float(np.finfo(dt).min)
    r = np.random.default_rng(2)
    rows = [np.full(V, -np.inf), np.full(V, low), np.zeros(V), np.where(np.arange(V) % 2, 0.0, -0.0), np.full(V, -3.5)]
    one = np.full(V, -np.inf); one[V - 1] = 4.0
    two = np.full(V, low); two[[1, V - 2]] = 0.0
    nan = r.normal(0, 1, V); nan[[3, V // 2]] = np.nan
    inf = r.normal(0, 1, V); inf[[5, V - 3]] = np.inf
    up, down = np.linspace(-9, 9, V), np.linspace(9, -9, V)
    steps = np.floor(np.arange(V) / 7.0) % 5
    certain = np.full(V, -30.0); certain[V // 3] = 30.0
    rows += [one, two, nan, inf, up, down, steps, certain, np.full(V, np.nan)]
    l = np.stack(rows).astype(dt)
    R = len(rows)
    for tokens in (np.zeros(R), np.full(R, V - 1), np.full(R, V // 3), np.full(R, 3), r.integers(0, V, R)):
        _check(l, tokens.astype(np.int32), min(32, V))
        _check(l, tokens.astype(np.int32), 3, 0.5, pad=1)


def test_logprobs_ties_take_the_lower_token():
    l = np.zeros((4, 5000), np.float32)
    l[1, [4999, 17, 300]] = 2.0
    l[2] = np.repeat(np.arange(50), 100)[::-1]
    l[3, 100:] = -0.0
    got = _check(l, np.array([4999, 300, 250, 99], np.int32), 5)
    assert got["top"][0].tolist() == [0, 1, 2, 3, 4] and got["rank"].tolist()[:2] == [4999, 1]


def test_logprobs_padding_tokens_and_partial_outputs():
    l, tokens = _rows(5, 6, 999, True)
    tokens[[0, 2, 3]] = [-1, 999, -2**31]
    got = _check(l, tokens, 4)
    assert got["logprob"][[0, 2, 3]].tolist() == [0, 0, 0] and got["rank"][[0, 2, 3]].tolist() == [-1, -1, -1]
    _check(l, None, 4)
    x, t = torch.from_numpy(l).cuda(), torch.from_numpy(tokens).cuda()
    lp, rank, h = torch.zeros(6, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda"), torch.zeros(6, device="cuda")
    ops.logprobs(x, t, lp, None, None, None, None)
    ops.logprobs(x, t, None, rank, None, None, None)
    ops.logprobs(x, None, None, None, h, None, None)
    torch.cuda.synchronize()
    assert (lp.cpu().numpy() == got["logprob"]).all() and (rank.cpu().numpy() == got["rank"]).all() and (h.cpu().numpy() == got["entropy"]).all()


def test_logprobs_rows_past_32_bit_offsets():
    """Rows whose element offsets pass 2^31: the last row of a buffer of 4.6 GB read through a wide row stride."""
    if torch.cuda.get_device_properties(0).total_memory < 12 << 30:
        pytest.skip("needs 12 GB")
    V, R = 1009, 5
    stride = (2**31 + 4096) // (R - 1)
    flat = torch.empty(stride * (R - 1) + V, dtype=torch.float16, device="cuda")
    x = flat.as_strided((R, V), (stride, 1))
    l, tokens = _rows(6, R, V, False)
    x.copy_(torch.from_numpy(l))
    o = [torch.zeros(R, device="cuda"), torch.zeros(R, dtype=torch.int32, device="cuda"), torch.zeros(R, device="cuda"),
         torch.zeros((R, 3), dtype=torch.int32, device="cuda"), torch.zeros((R, 3), device="cuda")]
    ops.logprobs(x, torch.from_numpy(tokens).cuda(), *o)
    torch.cuda.synchronize()
    want = refs.logprobs(l, tokens, 3, 1.0)
    assert (o[3].cpu().numpy() == want["top"]).all() and (o[1].cpu().numpy() == want["rank"]).all()
    assert np.abs(o[0].cpu().numpy() - want["logprob"]).max() < 1e-5


def test_logprobs_repeat_capture_and_two_streams():
    """The same bits every time, in a replayed graph that follows its input, and on two streams at once."""
    l, tokens = _rows(7, 40, 30011, True)
    l2, tokens2 = _rows(8, 40, 30011, True)
    first = _call(l, tokens, 20)
    first2 = _call(l2, tokens2, 20)
    x, t = torch.from_numpy(l).cuda(), torch.from_numpy(tokens).cuda()
    mk = lambda: [torch.zeros(40, device="cuda"), torch.zeros(40, dtype=torch.int32, device="cuda"), torch.zeros(40, device="cuda"),
                  torch.zeros((40, 20), dtype=torch.int32, device="cuda"), torch.zeros((40, 20), device="cuda")]
    same = lambda o, w: all((a.cpu().numpy() == w[k]).all() for a, k in zip(o, ("logprob", "rank", "entropy", "top", "top_logprob")))
    o = mk()
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        ops.logprobs(x, t, *o, stream=s)
    for v, tk, want in ((l, tokens, first), (l2, tokens2, first2), (l, tokens, first)):
        x.copy_(torch.from_numpy(v))
        t.copy_(torch.from_numpy(tk))
        g.replay()
        torch.cuda.synchronize()
        assert same(o, want)
    ins = [(torch.from_numpy(v).cuda(), torch.from_numpy(tk).cuda(), mk(), torch.cuda.Stream()) for v, tk in ((l, tokens), (l2, tokens2))]
    torch.cuda.synchronize()
    for _ in range(4):
        for xv, tv, ov, st in ins:
            ops.logprobs(xv, tv, *ov, stream=st)
    torch.cuda.synchronize()
    assert same(ins[0][2], first) and same(ins[1][2], first2)


def test_logprobs_refuses_tensors_that_do_not_fit():
    x = torch.zeros((3, 50), device="cuda")
    t = torch.zeros(3, dtype=torch.int32, device="cuda")
    lp, rank = torch.zeros(3, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    ti, tl = torch.zeros((3, 4), dtype=torch.int32, device="cuda"), torch.zeros((3, 4), device="cuda")
    good = dict(logits=x, tokens=t, logprob=lp, rank=rank, entropy=None, top_idx=ti, top_logprob=tl)
    wide = (torch.zeros((3, 33), dtype=torch.int32, device="cuda"), torch.zeros((3, 33), device="cuda"))
    for bad in (dict(tokens=t.long()), dict(tokens=t[:2]), dict(tokens=None), dict(logprob=lp.half()), dict(rank=rank.long()), dict(top_idx=None),
                dict(top_idx=ti[:, :2]), dict(top_logprob=tl.t()), dict(vocab=51), dict(vocab=0), dict(vocab=3), dict(inv_temp=0.0),
                dict(inv_temp=float("nan")), dict(inv_temp=float("inf")), dict(logits=x.double()), dict(logits=x.t()), dict(logits=x.cpu()),
                dict(top_idx=wide[0], top_logprob=wide[1]), dict(logits=x[:, ::2]),
                dict(tokens=None, logprob=None, rank=None, top_idx=None, top_logprob=None)):
        with pytest.raises(Error):
            ops.logprobs(**{**good, **bad})

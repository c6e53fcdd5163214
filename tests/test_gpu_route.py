"""Routing to experts against the definition in 64 bits: indices equal, weights within the rounding of fp32."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from berth_b200 import Error, kernels, moe, synth   # noqa: E402
from tests import operator_refs as refs   # noqa: E402
from tests.gpu_util import MAX_REL, MEAN_REL, dev, rel_errors   # noqa: E402


def _make(seed, T, E, f32=True, bias=True):
    r = np.random.default_rng(seed)
    popular = r.normal(0, 0.5, E)
    l = (r.normal(0, 1, (T, E)) + popular).astype(np.float32 if f32 else np.float16)
    return l, (-0.2 * popular + r.normal(0, 0.02, E)).astype(np.float32) if bias else None


def _run(l, bias, k, score="softmax", groups=1, keep=1, group_score="max", renorm=True, scale=1.0, pad=0, stream=None):
    T, E = l.shape
    wide = torch.full((T, E + pad), float("nan"), dtype=torch.float32 if l.dtype == np.float32 else torch.float16, device="cuda")
    wide[:, :E] = torch.from_numpy(l).cuda()
    idx = torch.full((T + 1, k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((T + 1, k), -7.0, dtype=torch.float32, device="cuda")
    b = None if bias is None else torch.from_numpy(bias).cuda()
    torch.cuda.synchronize()
    moe.route(wide[:, :E], b, idx[:T], w[:T], k, score=score, n_group=groups, topk_group=keep, group_score=group_score, renormalize=renorm, scale=scale,
              stream=stream)
    torch.cuda.synchronize()
    assert (idx[T] == -7).all() and (w[T] == -7.0).all()         # the row behind the last token is left as it was
    return idx[:T].cpu().numpy(), w[:T].cpu().numpy()


def _check(l, bias, k, **kw):
    idx, w = _run(l, bias, k, **kw)
    want_idx, want_w = refs.route(l, bias, k, kw.get("score", "softmax"), kw.get("groups", 1), kw.get("keep", 1), kw.get("group_score", "max"),
                                  kw.get("renorm", True), kw.get("scale", 1.0))
    assert (idx == want_idx).all(), np.argwhere(idx != want_idx)[:4]
    fin = np.isfinite(l)
    spread = float(np.minimum(np.where(fin, l, -np.inf).max(initial=-1e30) - np.where(fin, l, np.inf).min(initial=1e30), 200.0)) if fin.any() else 0.0
    # exp's argument is rounded once (half a step of at most the logits' spread; sigmoid: of the logit), exp and the division are
    # off by at most 2 and 1 steps, the sum of up to 1024 terms by 32 + 5 half steps along its longest path
    tol = (max(spread, np.abs(l[fin]).max(initial=0.0) if spread < 200 else 200.0) + 64) * 2.0 ** -24
    assert (np.isnan(w) == np.isnan(want_w)).all()
    ok = np.abs(w - want_w) <= tol * np.abs(want_w) + 1e-37
    assert (ok | np.isnan(want_w)).all(), (w[~ok][:4], want_w[~ok][:4])
    return idx, w


SHAPES = [(1, 256, 8, 1, 1, "max"), (5, 256, 8, 8, 4, "top2"), (129, 160, 6, 8, 3, "max"), (3, 7, 7, 1, 1, "max"), (9, 33, 3, 3, 2, "top2"),
          (4, 1024, 32, 1, 1, "max"), (2, 1023, 17, 3, 1, "top2"), (33, 300, 6, 4, 3, "top2"), (6, 64, 8, 32, 8, "top2"), (5, 32, 4, 32, 9, "max"),
          (7, 1, 1, 1, 1, "max"), (64, 512, 10, 8, 8, "top2"), (3, 130, 2, 13, 2, "max"), (2, 992, 30, 31, 5, "top2"), (257, 128, 8, 1, 1, "max")]


@pytest.mark.parametrize("T,E,k,groups,keep,gs", SHAPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("f32", [True, False])
def test_route_against_the_definition(T, E, k, groups, keep, gs, score, bias, f32):
    l, b = _make(hash((T, E, k)) % 1000, T, E, f32, bias)
    for renorm, scale, pad in ((True, 1.0, 0), (False, 2.5, 3)):
        _check(l, b, k, score=score, groups=groups, keep=keep, group_score=gs, renorm=renorm, scale=scale, pad=pad)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep,gs", [(1, 1, "max"), (4, 2, "top2"), (4, 2, "max")])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("f32", [True, False])
def test_masked_infinite_and_equal_logits(score, groups, keep, gs, bias, f32):
    E, k = 64, 6
    r = np.random.default_rng(3)
    low = np.finfo(np.float32 if f32 else np.float16).min
    rows = [np.full(E, -np.inf), np.full(E, low), np.zeros(E), np.full(E, 5.0)]
    one = np.full(E, -np.inf); one[37] = 0.25
    few = np.full(E, -np.inf); few[[3, 20, 21, 50]] = [1.0, 1.0, -2.0, 1.0]
    lowest = r.normal(0, 1, E); lowest[::2] = low
    half = r.normal(0, 1, E); half[::2] = -np.inf
    high = r.normal(0, 1, E); high[[5, 9]] = np.inf
    far = r.normal(-60, 10, E)
    steps = np.repeat(np.arange(8), 8)[::-1] * 0.5
    rows += [one, few, lowest, half, high, far, steps]
    l = np.stack(rows).astype(np.float32 if f32 else np.float16)
    b = r.normal(0, 0.1, E).astype(np.float32) if bias else None
    for renorm in (True, False):
        idx, w = _check(l, b, k, score=score, groups=groups, keep=keep, group_score=gs, renorm=renorm)
        assert (w[0] == 0).all() and len(set(idx[0])) == k
        if not bias:
            assert (idx[0] == np.arange(k)).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("renorm", [True, False])
def test_nan_logits_give_valid_indices_and_nan_weights(score, groups, renorm):
    E, k = 64, 8
    l, b = _make(4, 4, E)
    l[0] = np.nan
    l[1, 1::2] = np.nan
    l[2, 63] = np.nan
    for bias in (None, b):
        idx, w = _check(l, bias, k, score=score, groups=groups, keep=max(1, groups // 2), renorm=renorm)
        for t in range(4):
            assert len(set(idx[t].tolist())) == k and idx[t].min() >= 0 and idx[t].max() < E
        assert np.isnan(w[:3]).all() and np.isfinite(w[3]).all()
        assert (idx[0] == np.arange(k)).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep,gs", [(1, 1, "max"), (8, 3, "top2"), (8, 3, "max")])
def test_choice_scores_closer_than_32_bits_tell_apart(score, groups, keep, gs):
    """Experts whose scores differ by about 1e-9 under a bias of equal size: the choice follows the difference, not the index."""
    r = np.random.default_rng(8)
    T, E, k = 40, 256, 8
    l = (0.5 + 1e-6 * r.integers(-30, 31, (T, E))).astype(np.float32)
    for size in (0.0, 1.0, 100.0):
        _check(l, np.full(E, size, np.float32), k, score=score, groups=groups, keep=keep, group_score=gs)
    _check(l, None, k, score=score, groups=groups, keep=keep, group_score=gs)


@pytest.mark.parametrize("T", [1, 5000])
def test_many_tokens_every_choice_equal(T):
    """Near ties turn up among many tokens; vectorised reference."""
    E, k, G, keep = 256, 8, 8, 4
    l, b = _make(11, T, E)
    idx, w = _run(l, b, k, score="sigmoid", groups=G, keep=keep, group_score="top2", scale=2.5)
    s = 1.0 / (1.0 + np.exp(-l.astype(np.float64)))
    c = s + b.astype(np.float64)
    worth = np.sort(c.reshape(T, G, -1), axis=2)[:, :, -2:].sum(2)
    kept = np.argsort(-worth, axis=1, kind="stable")[:, :keep]
    allowed = np.zeros((T, G), bool)
    np.put_along_axis(allowed, kept, True, 1)
    want = np.argsort(-np.where(np.repeat(allowed, E // G, 1), c, -np.inf), axis=1, kind="stable")[:, :k]
    assert (idx == want).all()
    sel = np.take_along_axis(s, want, 1)
    assert np.allclose(w, 2.5 * sel / sel.sum(1, keepdims=True), rtol=80 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("groups,keep,gs", [(1, 1, "max"), (4, 3, "top2"), (4, 2, "max")])
@pytest.mark.parametrize("E,f32", [(88, True), (88, False), (256, True), (320, True)])
def test_many_tokens_softmax_under_a_bias(groups, keep, gs, E, f32):
    """Scores and bias of one size, so that of thousands of tokens some have neighbours that 32 bits cannot tell; a vectorised
    reference.  Half of the tokens are sharp: there the scores' errors are those of values near 1."""
    T, k = 6000, 9
    r = np.random.default_rng(E + groups)
    l = r.normal(0, 1, (T, E)) * np.where(np.arange(T) % 2, 4.0, 1.0)[:, None]
    l = l.astype(np.float32 if f32 else np.float16)
    b = (r.normal(0, 0.5, E) / E).astype(np.float32)
    idx, _ = _run(l, b, k, score="softmax", groups=groups, keep=keep, group_score=gs, scale=1.0)
    x = l.astype(np.float64)
    s = np.exp(x - x.max(1, keepdims=True))
    c = s / s.sum(1, keepdims=True) + b.astype(np.float64)
    best = np.sort(c.reshape(T, groups, -1), axis=2)
    worth = best[:, :, -2:].sum(2) if gs == "top2" else best[:, :, -1]
    kept = np.argsort(-worth, axis=1, kind="stable")[:, :keep]
    allowed = np.zeros((T, groups), bool)
    np.put_along_axis(allowed, kept, True, 1)
    want = np.argsort(-np.where(np.repeat(allowed, E // groups, 1), c, -np.inf), axis=1, kind="stable")[:, :k]
    assert (idx == want).all()


def test_route_captured_and_on_two_streams():
    """A captured and replayed call follows its inputs; two streams at once share nothing."""
    l, b = _make(21, 300, 128)
    l2, _ = _make(22, 300, 128)
    want, want2 = (refs.route(v, b, 4, "sigmoid", 4, 2, "top2", True, 1.0)[0] for v in (l, l2))
    x, bias = torch.from_numpy(l).cuda(), torch.from_numpy(b).cuda()
    idx, w = torch.zeros((300, 4), dtype=torch.int32, device="cuda"), torch.zeros((300, 4), device="cuda")
    kw = dict(score="sigmoid", n_group=4, topk_group=2, group_score="top2")
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        moe.route(x, bias, idx, w, 4, stream=s, **kw)
    for v, wanted in ((l, want), (l2, want2), (l, want)):
        x.copy_(torch.from_numpy(v))
        g.replay()
        torch.cuda.synchronize()
        assert (idx.cpu().numpy() == wanted).all()
    outs = []
    for v in (l, l2):
        st, xv = torch.cuda.Stream(), torch.from_numpy(v).cuda()
        o = (torch.zeros((300, 4), dtype=torch.int32, device="cuda"), torch.zeros((300, 4), device="cuda"))
        torch.cuda.synchronize()
        for _ in range(5):
            moe.route(xv, bias, *o, 4, stream=st, **kw)
        outs.append((o, xv))
    torch.cuda.synchronize()
    assert (outs[0][0][0].cpu().numpy() == want).all() and (outs[1][0][0].cpu().numpy() == want2).all()


ROUTINGS = [dict(score="sigmoid", n_group=4, topk_group=2, group_score="top2", renormalize=True, scale=2.5),
            dict(score="softmax", n_group=8, topk_group=3, renormalize=False, scale=4.0), dict(score="sigmoid", renormalize=False)]


def _want(oracle, wts, x, r, bias):
    logits = oracle.router_logits(x, wts["w_router"], wts["router_bias"])
    return refs.route(logits, bias, wts["top_k"], r["score"], r.get("n_group", 1), r.get("topk_group", 1), r.get("group_score", "max"),
                      r.get("renormalize", True), r.get("scale", 1.0))


@pytest.mark.parametrize("r", ROUTINGS)
@pytest.mark.parametrize("T", [1, 5, 130])
@pytest.mark.parametrize("shared", [0, 128])
def test_moe_layer_with_routing_vs_oracle(oracle, r, T, shared):
    H, I, E, k = 256, 128, 32, 4
    wts = synth.moe_layer_weights(1234, "rt", H, I, E, k, 4, 2, shared_inter=shared)
    bias = np.random.default_rng(5).normal(0, 0.1, E).astype(np.float32)
    x = synth.activations(1234, f"rt.x{T}", T, H)
    layer = moe.MoeLayer(torch.device("cuda"), wts, T, routing=moe.Routing(selection_bias=bias, **r))
    out = torch.full((T, H), float("nan"), dtype=torch.float32, device="cuda")
    idx = torch.empty((T, k), dtype=torch.int32, device="cuda")
    w = torch.empty((T, k), dtype=torch.float32, device="cuda")
    layer.forward(dev(x), out, idx, w)
    torch.cuda.synchronize()
    assert kernels.device_status(torch.cuda.current_device()) == 0
    assert "k_moe_route<" in moe.last_launch() and "k_moe_topk" not in moe.last_launch()
    want_idx, want_w = _want(oracle, wts, x, r, bias)
    assert (idx.cpu().numpy() == want_idx).all()
    assert np.allclose(w.cpu().numpy(), want_w, rtol=80 * 2.0 ** -24, atol=0)
    y64 = oracle.moe_layer_f64(wts, x, want_idx.astype(np.int32), want_w.astype(np.float32))
    mx, mean = rel_errors(out.cpu().numpy(), y64)
    assert mx <= MAX_REL and mean <= MEAN_REL, (mx, mean)


def test_stages_and_expert_parallel_sends_route_alike(oracle):
    """GpuStages.route, ep_send and the peer-memory send of one rank choose what berth_moe_layer_routed chooses."""
    import ctypes as C
    from berth_b200 import _lib
    H, I, E, k, T = 256, 128, 32, 4, 24
    wts = synth.moe_layer_weights(1234, "rt", H, I, E, k, 4, 2, shared_inter=128)
    bias = np.random.default_rng(5).normal(0, 0.1, E).astype(np.float32)
    x = synth.activations(1234, "rt.ep", T, H)
    r = ROUTINGS[0]
    want_idx, want_w = _want(oracle, wts, x, r, bias)
    device = torch.device("cuda", torch.cuda.current_device())
    st = moe.GpuStages(device, wts, E, max_rows=T * k + T, max_rows_per_expert=T, routing=moe.Routing(selection_bias=torch.from_numpy(bias), **r))
    xd = dev(x)
    l = _lib.lib()
    z = lambda n, dt=torch.uint8: torch.zeros(n, dtype=dt, device=device)
    cnt, flags, recv = z(E * 4), z(3 * 8 * 4), z((T * k + T) * H * 2)
    ptrs = lambda t: (C.c_void_p * 1)(t.data_ptr())
    ws = z(l.berth_moe_p2p_send_workspace_bytes(T, E, k, 1))
    pi, pw, inv = z(T * k, torch.int32), z(T * k, torch.float32), z(T * k, torch.int32)
    rc = l.berth_moe_p2p_send_routed(xd.data_ptr(), T, st.layer._keep["w_router"].data_ptr(), None, st.routing, H, E, k, pi.data_ptr(), pw.data_ptr(),
                                     inv.data_ptr(), 0, 1, 1, ptrs(cnt), ptrs(flags), ptrs(recv), T * k + T, ws.data_ptr(), ws.numel(), None)
    assert rc == 0, moe.last_error()
    assert "k_moe_route<" in moe.last_launch()
    a = st.route(xd)
    b = st.ep_send(xd, T)[:2]
    assert "k_moe_route<" in moe.last_launch()
    torch.cuda.synchronize()
    assert kernels.device_status(torch.cuda.current_device()) == 0
    for idx, w in (a, b, (pi.view(T, k), pw.view(T, k))):
        assert (idx.cpu().numpy() == want_idx).all()
        assert np.allclose(w.cpu().numpy(), want_w, rtol=80 * 2.0 ** -24, atol=0)


def test_routing_none_is_the_layer_as_it_was():
    """berth_moe_layer_routed with no routing: bit for bit berth_moe_layer."""
    import ctypes as C
    from berth_b200 import _lib
    H, I, E, k, T = 256, 128, 32, 4, 9
    wts = synth.moe_layer_weights(1234, "rt", H, I, E, k, 4, 2, shared_inter=128)
    layer = moe.MoeLayer(torch.device("cuda"), wts, T)
    x = dev(synth.activations(1234, "rt.none", T, H))
    got = []
    for old in (True, False):
        out = torch.empty((T, H), dtype=torch.float32, device="cuda")
        idx, w = torch.empty((T, k), dtype=torch.int32, device="cuda"), torch.empty((T, k), device="cuda")
        if old:
            assert _lib.lib().berth_moe_layer(C.byref(layer.c), x.data_ptr(), T, out.data_ptr(), idx.data_ptr(), w.data_ptr(),
                                              layer.workspace.data_ptr(), layer.workspace.numel(), None) == 0
        else:
            layer.forward(x, out, idx, w)
        torch.cuda.synchronize()
        assert "k_moe_topk" in moe.last_launch()
        got.append((out, idx, w))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_route_refuses_tensors_that_do_not_fit():
    l, b = _make(1, 4, 32)
    x = torch.from_numpy(l).cuda()
    idx, w = torch.empty((4, 2), dtype=torch.int32, device="cuda"), torch.empty((4, 2), device="cuda")
    for bad in (dict(topk_idx=idx.long()), dict(topk_idx=idx[:3]), dict(topk_w=w.half()), dict(logits=x.double()), dict(logits=x.t()),
                dict(selection_bias=torch.zeros(31, device="cuda")), dict(selection_bias=torch.zeros(32)), dict(top_k=3), dict(n_group=5),
                dict(score="tanh"), dict(group_score="mean"), dict(n_group=4, topk_group=5), dict(n_group=32, topk_group=1, group_score="max")):
        args = dict(logits=x, selection_bias=None, topk_idx=idx, topk_w=w, top_k=2)
        args.update(bad)
        with pytest.raises(Error):
            moe.route(**args)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep,gs", [(1, 1, "max"), (8, 3, "top2"), (8, 3, "max")])
@pytest.mark.parametrize("size", [2.0**25, 2.0**27, -2.0**33, 1e10, -1e12, 1e20, 3e38])
def test_biases_that_swallow_the_scores(score, groups, keep, gs, size):
    """A bias of which 64 bits leave few or none of a score's: choice scores that are equal there are ties, for the lower expert.  One
    bias for all, two sizes, and the large one for every other expert (a mask by bias)."""
    T, E, k = 24, 256, 8
    l, b = _make(31, T, E)
    for bias in (np.full(E, size), size * (1 + np.arange(E) // 64 % 2 * 2.0**-20), np.where(np.arange(E) % 2, size, b)):
        _check(l, bias.astype(np.float32), k, score=score, groups=groups, keep=keep, group_score=gs)


@pytest.mark.parametrize("rank", [0, 1])
def test_stages_of_one_rank_choose_among_all_ranks_experts(oracle, rank):
    """GpuStages that hold half of the layer's experts: the bias and the groups are those of all of them."""
    H, I, E, k, T = 256, 128, 32, 4, 24
    wts = synth.moe_layer_weights(1234, "rt", H, I, E, k, 4, 2, shared_inter=128)
    bias = np.random.default_rng(6).normal(0, 0.1, E).astype(np.float32)
    x = synth.activations(1234, "rt.half", T, H)
    half = {**wts, "n_experts": E // 2}
    for name in ("gate", "up", "down"):
        for part in ("trellis", "suh", "svh"):
            half[f"{name}_{part}"] = wts[f"{name}_{part}"][rank * E // 2:(rank + 1) * E // 2]
    device = torch.device("cuda", torch.cuda.current_device())
    for r in ROUTINGS:
        want_idx, want_w = _want(oracle, wts, x, r, bias)
        assert (want_idx < E // 2).any() and (want_idx >= E // 2).any()
        st = moe.GpuStages(device, half, E, max_rows=T * k + T, max_rows_per_expert=T, routing=moe.Routing(selection_bias=bias, **r))
        xd = dev(x)
        idx, w, inv, rows, counts = st.ep_send(xd, T)
        torch.cuda.synchronize()
        for i, v in ((idx, w), st.route(xd)):
            assert (i.cpu().numpy() == want_idx).all()
            assert np.allclose(v.cpu().numpy(), want_w, rtol=80 * 2.0 ** -24, atol=0)
        assert (counts.cpu().numpy() == np.bincount(want_idx.ravel(), minlength=E)).all()
        assert torch.equal(rows[inv.long()].view(torch.int16), xd.repeat_interleave(k, 0).view(torch.int16))
    assert kernels.device_status(torch.cuda.current_device()) == 0

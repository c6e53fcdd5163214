"""Rotary positions against the definition in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from berth_b200 import Error, kernels   # noqa: E402
from berth_b200.kernels import ops   # noqa: E402
from tests import operator_refs as refs   # noqa: E402

EPS, BIAS = 1e-6, 1.0


def _layout(T, H, D, dt, kind, r):
    """A [T][H][D] view: "plain", columns of a wider buffer, a gate behind each head, heads outside tokens (a cache), or shifted by
    one element so that no row is aligned."""
    if kind == "packed":
        return torch.zeros((T, H + 3, D), dtype=dt, device="cuda")[:, 1:H + 1]
    if kind == "gated":
        return torch.zeros((T, H, 2 * D), dtype=dt, device="cuda")[:, :, :D]
    if kind == "cache":
        return torch.zeros((H, T + 2, D), dtype=dt, device="cuda")[:, :T].transpose(0, 1)
    if kind == "shifted":
        return torch.zeros(T * H * D + 1, dtype=dt, device="cuda")[1:].view(T, H, D)
    return torch.zeros((T, H, D), dtype=dt, device="cuda")


def _case(seed, T, hq, hk, D, rot, dt, norm, far=0, base=1e4):
    r = np.random.default_rng(seed)
    x = [torch.from_numpy(r.normal(0, 1, (T, h, D))).to(dt) for h in (hq, hk)]
    pos = r.integers(0, 5000, T) + far
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    norms = [torch.from_numpy(r.normal(0, 0.1, D)).bfloat16() if norm else None for _ in range(2)]
    return x, pos.astype(np.int32), np.array(f), norms


def _check(x, pos, f, norms, interleaved, factor=1.0, kinds=("plain", "plain"), in_place=False, stream=None):
    ins = []
    for t in x:
        v = _layout(*t.shape, t.dtype, kinds[0], None)
        v.copy_(t)
        ins.append(v)
    outs = ins if in_place else [_layout(*t.shape, t.dtype, kinds[1], None) for t in x]
    nd = [None if n is None else n.cuda() for n in norms]
    inv = torch.tensor(f, dtype=torch.float64, device="cuda")
    p = torch.from_numpy(pos).cuda()
    bases = [o._base if o._base is not None else o for o in outs]
    before = [b.clone() for b in bases]
    torch.cuda.synchronize()
    ops.rope(ins[0], ins[1], p, inv, outs[0], outs[1], interleaved, factor, nd[0], nd[1], EPS, BIAS, stream=stream)
    torch.cuda.synchronize()
    for t, o, n, b, was in zip(x, outs, norms, bases, before):
        n64 = None if n is None else n.double().numpy()
        want, size = refs.rope(t.numpy(), pos, f, interleaved, factor, n64, EPS, BIAS)
        got = o.cpu().double().numpy()
        # fp32 inside: the angle to 2^-25 of a turn (1.9e-7), cos and sin to 2 steps of at most 2^-24, the factor, two products
        # and a sum half a step each: below 2^-20 of |x_a| + |x_b|; the norm's sum of squares, root, division and two products
        # another (512 / 32 + 5) / 2 + 6 half steps; then the output's own rounding
        eps32 = 2.0 ** -20 + (17 * 2.0 ** -24 if n is not None else 0.0)
        half_step = torch.finfo(t.dtype).eps / 2
        tol = size * eps32 + np.abs(want) * half_step + (2.0 ** -25 if t.dtype == torch.float16 else 0.0)
        bad = np.abs(got - want) > tol
        assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])
        if n is None:      # what does not turn is passed on bit for bit
            assert (got[..., 2 * len(f):] == t.double().numpy()[..., 2 * len(f):]).all()
        # nothing beside the outputs changed
        touched = torch.zeros_like(b, dtype=torch.bool)
        touched.as_strided(o.shape, o.stride(), o.storage_offset()).fill_(True)
        assert torch.equal(b[~touched], was[~touched])


DIMS = [(64, 64), (128, 128), (256, 64), (256, 256), (80, 80), (96, 48), (128, 88), (128, 2), (66, 34), (7, 6), (512, 512), (40, 26), (192, 64)]


@pytest.mark.parametrize("D,rot", DIMS)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_rope_against_the_definition(D, rot, interleaved, norm, dt):
    for T, hq, hk in ((1, 24, 4), (3, 1, 1), (37, 5, 2)):
        x, pos, f, norms = _case(T + D, T, hq, hk, D, rot, dt, norm)
        _check(x, pos, f, norms, interleaved, factor=1.0 if T == 3 else 1.3465735902799727)


@pytest.mark.parametrize("kinds", [("packed", "plain"), ("gated", "plain"), ("plain", "cache"), ("shifted", "plain"), ("plain", "shifted"),
                                   ("cache", "gated")])
@pytest.mark.parametrize("D,rot", [(128, 128), (256, 64), (80, 26)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_rope_strides(kinds, D, rot, interleaved, norm):
    for dt in (torch.float16, torch.float32):
        x, pos, f, norms = _case(9, 19, 6, 2, D, rot, dt, norm)
        _check(x, pos, f, norms, interleaved, kinds=kinds)


@pytest.mark.parametrize("kind", ["plain", "packed", "gated", "cache", "shifted"])
@pytest.mark.parametrize("D,rot", [(128, 128), (256, 64), (128, 40), (72, 34), (512, 480)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_rope_in_place(kind, D, rot, interleaved, norm):
    x, pos, f, norms = _case(13, 21, 7, 3, D, rot, torch.float16, norm)
    _check(x, pos, f, norms, interleaved, kinds=(kind, kind), in_place=True)


@pytest.mark.parametrize("D,rot", [(80, 40), (128, 88), (256, 8), (80, 36), (128, 92), (512, 508), (80, 12), (80, 38), (128, 42), (24, 2), (8, 8), (16, 6)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_rope_pieces(D, rot, interleaved, norm, dt):
    """Every width of the pieces (16, 8, 4 bytes and none), by what half of the rotated part is a multiple of; what is passed on may be
    infinite where no norm takes it in."""
    x, pos, f, norms = _case(51, 53, 9, 2, D, rot, dt, norm)
    if not norm and rot < D:
        for t in x:
            t[::3, :, rot] = float("inf")
            t[1::3, 1:, D - 1] = float("-inf")
    _check(x, pos, f, norms, interleaved, factor=0.75)
    half = rot // 2 * x[0].element_size()
    want = 16 if interleaved or half % 16 == 0 else 8 if half % 8 == 0 else 4 if half % 4 == 0 else 0
    assert ops.last_launch().endswith(f" piece={want}") and ops.last_launch().startswith("k_rope_any") == (want == 0)
    _check(x, pos, f, norms, interleaved, kinds=("gated", "packed"))
    _check(x, pos, f, norms, interleaved, kinds=("shifted", "plain"))
    _check(x, pos, f, norms, interleaved, kinds=("cache", "cache"), in_place=True)


@pytest.mark.parametrize("T,early", [(4001, False), (500, True)])
@pytest.mark.parametrize("D,rot,interleaved", [(128, 128, False), (80, 40, False), (128, 92, False), (80, 38, False), (96, 90, True)])
@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_rope_norms_of_few_and_many_blocks(T, early, D, rot, interleaved, dt):
    """The two ways to read the norm's weights."""
    x, pos, f, norms = _case(T + rot, T, 6, 1, D, rot, dt, True)
    _check(x, pos, f, norms, interleaved)
    assert ("early" in ops.last_launch()) == (early and "any" not in ops.last_launch())
    _check(x, pos, f, [norms[0], None], interleaved, kinds=("packed", "gated"))


@pytest.mark.parametrize("dt", [torch.float16, torch.float32])
def test_rope_far_and_negative_positions(dt):
    """Positions whose angle needs more than 32 bits, the largest and the most negative one."""
    x, pos, f, norms = _case(17, 9, 4, 2, 128, 128, dt, False, base=1e6)
    for pos in (pos + 1_000_000, np.array([0, -1, 2**31 - 1, -2**31, 123456789, 1, 2**30, -77, 2**24 + 1]).astype(np.int32)):
        _check(x, pos, f, norms, False)


def test_rope_many_tokens_and_heads():
    x, pos, f, norms = _case(23, 1500, 32, 8, 128, 128, torch.float16, False)
    _check(x, pos, f, norms, False, kinds=("packed", "plain"))
    x, pos, f, norms = _case(24, 700, 24, 4, 256, 64, torch.float16, True)
    _check(x, pos, f, norms, False, kinds=("gated", "plain"))
    x, pos, f, norms = _case(25, 2, 1024, 1024, 64, 64, torch.float32, False)
    _check(x, pos, f, norms, True)


def test_rope_without_k_and_one_norm():
    x, pos, f, norms = _case(31, 5, 4, 2, 64, 64, torch.float16, True)
    q, k, out_q, out_k = x[0].cuda(), x[1].cuda(), torch.zeros_like(x[0], device="cuda"), torch.zeros_like(x[1], device="cuda")
    p, inv, n = torch.from_numpy(pos).cuda(), torch.tensor(f, dtype=torch.float64, device="cuda"), norms[0].cuda()
    alone = torch.zeros_like(out_q)
    ops.rope(q, k, p, inv, out_q, out_k, q_norm=n, norm_epsilon=EPS, norm_bias=BIAS)
    ops.rope(q, None, p, inv, alone, None, q_norm=n, norm_epsilon=EPS, norm_bias=BIAS)
    bare = torch.zeros_like(out_k)
    ops.rope(k, None, p, inv, bare, None)
    torch.cuda.synchronize()
    assert torch.equal(out_q, alone) and torch.equal(out_k, bare)


def test_rope_zero_rows_with_norm():
    """A head of zeros: r = 1 / sqrt(eps), the output zero."""
    q = torch.zeros((2, 3, 64), dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 5.0)
    ops.rope(q, None, torch.tensor([1, 2], dtype=torch.int32, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda"), out, None,
             q_norm=torch.ones(64, dtype=torch.bfloat16, device="cuda"))
    torch.cuda.synchronize()
    assert (out == 0).all()


def test_rope_captured_and_on_two_streams():
    x, pos, f, norms = _case(41, 64, 8, 2, 128, 128, torch.float16, True)
    q, k = x[0].cuda(), x[1].cuda()
    p, inv = torch.from_numpy(pos).cuda(), torch.tensor(f, dtype=torch.float64, device="cuda")
    n = [v.cuda() for v in norms]
    eager = [torch.zeros_like(q), torch.zeros_like(k)]
    graphed = [torch.zeros_like(q), torch.zeros_like(k)]
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        ops.rope(q, k, p, inv, graphed[0], graphed[1], False, 1.0, n[0], n[1], EPS, BIAS, stream=s)
    for shift in (0, 7):
        p += shift
        ops.rope(q, k, p, inv, eager[0], eager[1], False, 1.0, n[0], n[1], EPS, BIAS)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, graphed))
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.zeros_like(q), torch.zeros_like(k)] for _ in streams]
    torch.cuda.synchronize()
    for _ in range(5):
        for st, o in zip(streams, outs):
            ops.rope(q, k, p, inv, o[0], o[1], False, 1.0, n[0], n[1], EPS, BIAS, stream=st)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(eager, o))


def test_rope_refuses_tensors_that_do_not_fit():
    q = torch.zeros((3, 4, 64), dtype=torch.float16, device="cuda")
    k = torch.zeros((3, 2, 64), dtype=torch.float16, device="cuda")
    p, inv = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda")
    good = dict(q=q, k=k, positions=p, inv_freq=inv, q_out=torch.empty_like(q), k_out=torch.empty_like(k))
    bads = [dict(positions=p.long()), dict(positions=p[:2]), dict(inv_freq=inv.float()), dict(inv_freq=torch.ones(33, dtype=torch.float64, device="cuda")),
            dict(q_out=torch.empty_like(q).float()), dict(q_out=torch.empty_like(k)), dict(k=None), dict(k=k.float()), dict(q=q[:, :, ::2]),
            dict(q=q.cpu()), dict(q_norm=torch.ones(64, device="cuda")), dict(q_norm=torch.ones(32, dtype=torch.bfloat16, device="cuda")),
            dict(q_out=torch.empty((3, 1, 64), dtype=torch.float16, device="cuda").expand(3, 4, 64)),
            dict(q_out=torch.empty((1, 4, 64), dtype=torch.float16, device="cuda").expand(3, 4, 64)),
            dict(q=q[:0], q_out=q[:0], k=k[:0], k_out=k[:0], positions=p[:0])]
    for bad in bads:
        with pytest.raises(Error):
            ops.rope(**{**good, **bad})

"""The cases of test_gpu_rope.py under a comparison that no NaN passes, into outputs that begin as NaN: an element that was not written,
or came out of a register that was not set, is wrong here."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from berth_b200.kernels import ops   # noqa: E402
from tests import operator_refs as refs   # noqa: E402
from tests import test_gpu_rope as cases   # noqa: E402
from tests.strict import wrong   # noqa: E402

EPS, BIAS = cases.EPS, cases.BIAS


def _layout(*a):
    v = cases_layout(*a)
    (v._base if v._base is not None else v).fill_(float("nan"))
    return v


def _check(x, pos, f, norms, interleaved, factor=1.0, kinds=("plain", "plain"), in_place=False, stream=None):
    """As in test_gpu_rope.py, with the tolerances that are derived there."""
    ins = []
    for t in x:
        v = _layout(*t.shape, t.dtype, kinds[0], None)
        v.copy_(t)
        ins.append(v)
    outs = ins if in_place else [_layout(*t.shape, t.dtype, kinds[1], None) for t in x]
    nd = [None if n is None else n.cuda() for n in norms]
    inv, p = torch.tensor(f, dtype=torch.float64, device="cuda"), torch.from_numpy(pos).cuda()
    bits = {torch.float16: torch.int16, torch.float32: torch.int32}[x[0].dtype]
    bases = [o._base if o._base is not None else o for o in outs]
    before = [b.clone() for b in bases]
    torch.cuda.synchronize()
    ops.rope(ins[0], ins[1], p, inv, outs[0], outs[1], interleaved, factor, nd[0], nd[1], EPS, BIAS, stream=stream)
    torch.cuda.synchronize()
    for t, o, n, b, was in zip(x, outs, norms, bases, before):
        want, size = refs.rope(t.numpy(), pos, f, interleaved, factor, None if n is None else n.double().numpy(), EPS, BIAS)
        got = o.cpu().double().numpy()
        eps32 = 2.0 ** -20 + (17 * 2.0 ** -24 if n is not None else 0.0)
        half_step = torch.finfo(t.dtype).eps / 2
        turned = np.zeros(t.shape[-1], bool)
        turned[:2 * len(f)] = True
        finite = np.isfinite(want)
        tol = np.where(finite, np.where(finite, size, 0) * eps32 + np.abs(np.where(finite, want, 0)) * half_step + (2.0 ** -25 if t.dtype == torch.float16 else 0.0), 0)
        if n is None:
            tol = np.where(turned, tol, 0.0)             # what does not turn is passed on as it is
        bad = wrong(got, want, tol)
        assert not bad.any(), (np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])
        touched = torch.zeros_like(b, dtype=torch.bool)  # nothing beside the outputs changed
        touched.as_strided(o.shape, o.stride(), o.storage_offset()).fill_(True)
        assert torch.equal(b.view(bits)[~touched], was.view(bits)[~touched])


cases_layout = cases._layout


@pytest.fixture(autouse=True)
def strictly(monkeypatch):
    monkeypatch.setattr(cases, "_check", _check)


test_against_the_definition = cases.test_rope_against_the_definition
test_strides = cases.test_rope_strides
test_in_place = cases.test_rope_in_place
test_pieces = cases.test_rope_pieces
test_norms_of_few_and_many_blocks = cases.test_rope_norms_of_few_and_many_blocks
test_far_and_negative_positions = cases.test_rope_far_and_negative_positions
test_many_tokens_and_heads = cases.test_rope_many_tokens_and_heads


def test_the_cases_run_under_this_comparison():
    assert cases._check is _check

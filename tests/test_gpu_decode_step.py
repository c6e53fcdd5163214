"""A decode step as a host runs it: q/k/v projections, rotary positions in place, output projection, experts chosen by a routing of the
layer's own, lm_head, log probabilities.  Every new step against its definition in 64 bits from the inputs that it really had, and
the whole step captured and replayed."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from berth_b200 import Codebook, OutDtype, kernels, moe, synth   # noqa: E402
from berth_b200.engine import Exl3Linear, Gpu, SlicedMultiLinear   # noqa: E402
from berth_b200.kernels import ops   # noqa: E402
from tests import operator_refs as refs   # noqa: E402

H, HEADS, KV, D, ROT, E, K, V = 256, 4, 2, 64, 32, 32, 4, 2048
EPS, BIAS = 1e-6, 1.0
ROUTING = dict(score="sigmoid", n_group=4, topk_group=2, group_score="top2", renormalize=True, scale=2.5)


class Step:
    def __init__(self, rows, stream=None):
        gpu = self.gpu = Gpu(torch.cuda.current_device(), stream)
        self.rows = rows
        r = np.random.default_rng(12)
        bf16 = lambda *s: torch.from_numpy(r.normal(0, 0.05, s)).bfloat16().cuda()
        lin = lambda name, k, n, bits=4: Exl3Linear(gpu, name, *(synth.linear_weights(77, name, k, n, bits)[p] for p in ("trellis", "suh", "svh")), bits,
                                                    Codebook.Mul1, max_rows=rows)
        # q with a gate behind each head
        self.qkv = SlicedMultiLinear(gpu, [lin("q", H, 2 * HEADS * D), lin("k", H, 2 * KV * D), lin("v", H, 2 * KV * D)], OutDtype.F16, max_rows=rows)
        self.o, self.head = lin("o", HEADS * D, H), lin("lm_head", H, V, 6)
        self.norms = [bf16(H) for _ in range(3)]
        self.q_norm, self.k_norm = bf16(D), bf16(D)
        f, self.factor = ops.rope_frequencies(ROT, 1e6, "yarn", factor=8.0, original_context=4096)
        self.inv_freq = torch.tensor(f, dtype=torch.float64, device="cuda")
        self.bias = r.normal(0, 0.1, E).astype(np.float32)
        self.moe = moe.MoeLayer(gpu.device, synth.moe_layer_weights(77, "moe", H, 128, E, K, 4, 2, shared_inter=128), rows,
                                routing=moe.Routing(selection_bias=self.bias, **ROUTING))
        z = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device="cuda")
        self.hidden, self.residual, self.x = z(rows, H), z(rows, H), z(rows, H, dt=torch.float16)
        self.position, self.attended = z(rows, dt=torch.int32), z(rows, HEADS * D, dt=torch.float16)
        self.q, self.k = z(rows, HEADS, D, dt=torch.float16), z(rows, 2 * KV, D, dt=torch.float16)
        self.mixed, self.idx, self.w = z(rows, H), z(rows, K, dt=torch.int32), z(rows, K)
        self.logits, self.best = z(rows, V), z(rows, dt=torch.int64)
        self.token, self.lp, self.rank, self.entropy = z(rows, dt=torch.int32), z(rows), z(rows, dt=torch.int32), z(rows)
        self.top, self.top_lp = z(rows, 5, dt=torch.int32), z(rows, 5)

    def run(self):
        gpu, rows, s = self.gpu, self.rows, self.gpu.raw_stream()
        self.residual.copy_(self.hidden)
        ops.rms_norm(self.residual, self.norms[0], self.x, rows, H, EPS, BIAS, 1.0, True, s)
        q, k, _ = self.qkv.forward_n(gpu, rows, self.x)
        self.q_in, self.k_in = q.view(rows, HEADS, 2 * D)[:, :, :D], k.view(rows, 2 * KV, D)
        ops.rope(self.q_in, self.k_in, self.position, self.inv_freq, self.q, self.k, False, self.factor, self.q_norm, self.k_norm, EPS, BIAS, stream=s)
        self.o.forward_n(gpu, rows, self.q, self.mixed, OutDtype.F32)        # (attention itself is the host's: q stands in)
        ops.rms_norm_res_in(self.mixed, self.norms[1], self.x, self.residual, rows, H, EPS, BIAS, 1.0, True, s)
        self.moe_in = self.x.clone()
        self.moe.forward(self.x, self.mixed, self.idx, self.w, gpu.stream)
        ops.rms_norm_res_in(self.mixed, self.norms[2], self.x, self.residual, rows, H, EPS, BIAS, 1.0, True, s)
        self.head.forward_argmax(gpu, rows, self.x, self.best, self.logits)
        # a key's low word is the token, complemented
        self.token.copy_(torch.bitwise_not(self.best.view(torch.int32).view(-1, 2)[:, 0]))
        ops.logprobs(self.logits, self.token, self.lp, self.rank, self.entropy, self.top, self.top_lp, V, 1.25, stream=s)

    def feed(self, seed):
        r = np.random.default_rng(seed)
        self.hidden.copy_(torch.from_numpy(r.normal(0, 1, (self.rows, H))).float())
        self.position.copy_(torch.from_numpy(r.integers(0, 100000, self.rows)).int())

    def outputs(self):
        return [t.clone() for t in (self.q, self.k, self.idx, self.w, self.logits, self.token, self.lp, self.rank, self.entropy, self.top, self.top_lp)]


@pytest.mark.parametrize("rows", [1, 3, 8])
def test_decode_step(oracle, rows):
    st = Step(rows)
    st.feed(rows)
    st.run()
    torch.cuda.synchronize()
    assert kernels.device_status(torch.cuda.current_device()) == 0
    f = st.inv_freq.cpu().numpy()
    for x, got, norm in ((st.q_in, st.q, st.q_norm), (st.k_in, st.k, st.k_norm)):
        want, size = refs.rope(x.cpu().numpy(), st.position.cpu().numpy(), f, False, st.factor, norm.double().cpu().numpy(), EPS, BIAS)
        assert (np.abs(got.cpu().double().numpy() - want) <= size * (2.0 ** -20 + 17 * 2.0 ** -24) + np.abs(want) * 2.0 ** -11 + 2.0 ** -25).all()
    wr = synth.moe_layer_weights(77, "moe", H, 128, E, K, 4, 2, shared_inter=128)["w_router"]
    logits = oracle.router_logits(st.moe_in.cpu().numpy(), wr)
    want_idx, want_w = refs.route(logits, st.bias, K, ROUTING["score"], 4, 2, "top2", True, 2.5)
    assert (st.idx.cpu().numpy() == want_idx).all() and np.allclose(st.w.cpu().numpy(), want_w, rtol=80 * 2.0 ** -24, atol=0)
    lg = st.logits.cpu().numpy()
    want = refs.logprobs(lg, st.token.cpu().numpy(), 5, 1.25)
    assert (st.token.cpu().numpy() == lg.argmax(1)).all() and (st.rank.cpu().numpy() == 0).all()
    assert (st.top.cpu().numpy() == want["top"]).all() and (st.top[:, 0] == st.token).all()
    tol = (V / 256 + 64) * 2.0 ** -24
    assert (np.abs(st.lp.cpu().numpy() - want["logprob"]) <= tol + np.abs(want["logprob"]) * 6 * 2.0 ** -24).all()
    assert (np.abs(st.top_lp.cpu().numpy() - want["top_logprob"]) <= tol + np.abs(want["top_logprob"]) * 6 * 2.0 ** -24).all()
    assert (np.abs(st.entropy.cpu().numpy() - want["entropy"]) <= 2 * tol * (1 + want["entropy"])).all()
    assert torch.equal(st.top_lp[:, 0], st.lp)


def test_decode_step_captured_and_replayed():
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        st = Step(2, stream)
        st.feed(1)
        st.run()                                  # what the library sets up once per device
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            st.run()
        for seed in (5, 6, 5):
            st.feed(seed)
            st.run()
            stream.synchronize()
            eager = st.outputs()
            for t in (st.q, st.k, st.idx, st.w, st.logits, st.lp, st.rank, st.entropy, st.top, st.top_lp):
                t.zero_()
            g.replay()
            stream.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(eager, st.outputs()))
    assert kernels.device_status(torch.cuda.current_device()) == 0

"""Expert parallelism under a routing of the layer's own, on CPU: a selection bias and groups over all ranks' experts, weights that do not
sum to one.  The exchange against the layer on one process."""
import os
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import torch.distributed as dist            # noqa: E402
import torch.multiprocessing as mp          # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
H, I, E, K, T = 128, 128, 8, 3, 6
ROUTINGS = [("sigmoid", 4, 2, "top2", True, 2.5), ("softmax", 4, 3, "max", False, 4.0), ("sigmoid", 2, 1, "top2", False, 1.0)]


def _bias():
    """Turns the choice to experts of both ranks that the scores alone would leave out."""
    return np.random.default_rng(3).normal(0, 0.3, E).astype(np.float32)


def _choose(orc, wts, x, routing):
    from tests import operator_refs as refs
    score, groups, keep, group_score, renorm, scale = routing
    idx, w = refs.route(orc.router_logits(x, wts["w_router"], wts.get("router_bias")), _bias(), K, score, groups, keep, group_score, renorm, scale)
    return idx.astype(np.int32), w.astype(np.float32)


def _worker(rank, world, port, tmp, which):
    sys.path.insert(0, ROOT)
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from berth_b200 import moe, synth
    from oracle import exl3_oracle as orc
    from tests.test_ep_gloo import OracleStages
    orc.set_num_threads(2)

    class Stages(OracleStages):
        def route(self, x):
            return tuple(torch.from_numpy(a) for a in _choose(self.orc, self.w, x.numpy(), ROUTINGS[which]))

        def sort(self, keys, e0, n_local, for_experts=False):
            perm, inv, offsets = super().sort(keys, e0, n_local)
            if for_experts:
                self._last_offsets = offsets.numpy()
            return perm, inv, offsets
    full = synth.moe_layer_weights(78, "ep", H, I, E, K, 4, 2, shared_inter=128)
    n_local = E // world
    local = {**full, "n_experts": n_local}
    for name in ("gate", "up", "down"):
        for part in ("trellis", "suh", "svh"):
            local[f"{name}_{part}"] = full[f"{name}_{part}"][rank * n_local:(rank + 1) * n_local]
    layer = moe.EpMoeLayer(Stages(local, rank * n_local, n_local, orc), dist.group.WORLD, E, K)
    x = synth.activations(78, "ep.x", T * world, H)[rank * T:(rank + 1) * T].copy()
    out, idx, w = layer.forward(torch.from_numpy(x))
    np.savez(os.path.join(tmp, f"{rank}.npz"), out=out.numpy(), idx=idx.numpy(), w=w.numpy())
    dist.destroy_process_group()


@pytest.mark.parametrize("which", range(len(ROUTINGS)))
def test_two_ranks_under_a_routing_match_one_process(oracle, tmp_path, which):
    world, port = 2, 29731 + (os.getpid() % 200)
    mp.spawn(_worker, args=(world, port, str(tmp_path), which), nprocs=world, join=True)
    from berth_b200 import synth
    full = synth.moe_layer_weights(78, "ep", H, I, E, K, 4, 2, shared_inter=128)
    x = synth.activations(78, "ep.x", T * world, H)
    want_idx, want_w = _choose(oracle, full, x, ROUTINGS[which])
    got = [np.load(tmp_path / f"{r}.npz") for r in range(world)]
    assert (np.concatenate([g["idx"] for g in got]) == want_idx).all()
    assert (np.concatenate([g["w"] for g in got]) == want_w).all()
    # experts of both ranks, and once (one group of two kept) every row on one rank
    assert {int(e) // (E // world) for e in want_idx.ravel()} == ({0} if which == 2 else {0, 1})
    y64 = oracle.moe_layer_f64(full, x, want_idx, want_w)
    out = np.concatenate([g["out"] for g in got])
    assert np.isfinite(out).all() and np.abs(out - y64).max() <= 1e-2 * np.sqrt((y64 ** 2).mean())

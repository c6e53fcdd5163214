"""Three operators that a decoder runs between its trellis linears, as cases for timing: the routing of tokens to
experts, rotary positions of q and k, and the log probabilities of an answer's tokens.

Each has its plain form in elementary torch operations here and, where ``own`` is true, the library's call.
"""
from __future__ import annotations

import math

import torch

own = False


def listed() -> list:
    groups = {"kind": "route", "score": "sigmoid", "bias": True, "experts": 256, "top_k": 8, "groups": 8, "keep": 4, "group_score": "top2",
              "renormalize": True, "scale": 2.5, "f32": True}
    a3b = {"kind": "rope", "q_heads": 24, "k_heads": 4, "dim": 256, "rot": 64, "interleaved": False, "norm": True, "layout": "gated", "base": 1e7,
           "scaling": "none", "far": 0, "f32": False}
    return [
        # one user's token chooses its experts: launch and latency count
        {"name": "route 1", "tokens": 1, **groups},
        # a decode batch, probabilities over all experts as weights
        {"name": "route 64", "kind": "route", "tokens": 64, "score": "softmax", "bias": False, "experts": 256, "top_k": 8, "groups": 1, "keep": 1,
         "group_score": "max", "renormalize": False, "scale": 1.0, "f32": True},
        # a ragged chunk behind a router whose logits are fp16, groups ranked by their best expert
        {"name": "route 1001", "kind": "route", "tokens": 1001, "score": "softmax", "bias": False, "experts": 160, "top_k": 6, "groups": 8, "keep": 3,
         "group_score": "max", "renormalize": False, "scale": 16.0, "f32": False},
        # the prefill chunk of a whole batch
        {"name": "route 16384", "tokens": 16384, **groups},
        # one user's token: q (with the gate of the attention's output behind each head) and k, normalised and rotated
        {"name": "rope 1", "tokens": 1, **a3b},
        # a decode batch in fp32, neighbouring pairs, positions of a context stretched by linear scaling
        {"name": "rope 32", "kind": "rope", "tokens": 32, "q_heads": 32, "k_heads": 8, "dim": 128, "rot": 128, "interleaved": True, "norm": False,
         "layout": "apart", "base": 1e4, "scaling": "linear", "far": 30000, "f32": True},
        # a short prompt's only chunk, of no round length
        {"name": "rope 421", "tokens": 421, **a3b},
        # a long prompt's chunk far into a stretched context, q/k/v in one buffer
        {"name": "rope 8192", "kind": "rope", "tokens": 8192, "q_heads": 32, "k_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "norm": False,
         "layout": "packed", "base": 1e6, "scaling": "yarn", "far": 900000, "f32": False},
        # the drawn token's log probability and twenty alternatives, one user
        {"name": "logprobs 1", "kind": "logprobs", "rows": 1, "vocab": 248320, "pad": 0, "top": 20, "temperature": 0.8, "masked": 0.0, "f32": True},
        # a decode batch whose rows are masked by a grammar
        {"name": "logprobs 32", "kind": "logprobs", "rows": 32, "vocab": 248320, "pad": 0, "top": 5, "temperature": 1.0, "masked": 0.3, "f32": True},
        # rows of an odd vocabulary in a padded buffer, scored without alternatives
        {"name": "logprobs 77", "kind": "logprobs", "rows": 77, "vocab": 100003, "pad": 29, "top": 0, "temperature": 1.0, "masked": 0.0, "f32": True},
        # every token of a prompt scored from fp16 logits
        {"name": "logprobs 421", "kind": "logprobs", "rows": 421, "vocab": 248320, "pad": 0, "top": 5, "temperature": 1.0, "masked": 0.0, "f32": False},
    ]


def _log(rng, lo: float, hi: float) -> int:
    """A whole number between lo and hi, spread over the logarithm."""
    return max(int(lo), min(int(hi), int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    """Any token count up to a full chunk, expert counts that groups divide or not, heads of 32 to 256 wide of which any
    even part turns, vocabularies of 1000 to 250000."""
    kind = rng.choice(["route", "rope", "logprobs"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        size = _log(rng, max(2, 8 // groups), 512 // groups)
        experts = groups * size
        keep = rng.randint((groups + 1) // 2, groups)
        return {"kind": kind, "tokens": _log(rng, 1, 16384 * min(1.0, 256 / experts)), "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5,
                "experts": experts, "top_k": rng.randint(1, min(10, keep * size)), "groups": groups, "keep": keep,
                "group_score": rng.choice(["max", "top2"]) if groups > 1 else "max", "renormalize": rng.random() < 0.6,
                "scale": rng.choice([1.0, 1.0, 2.5, 16.0]), "f32": rng.random() < 0.75}
    if kind == "rope":
        k_heads = rng.choice([1, 2, 4, 8])
        q_heads = k_heads * rng.randint(1, 8)
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        f32 = rng.random() < 0.25
        most = 8192 * 40 * 128 / ((q_heads + k_heads) * dim * (2 if f32 else 1))
        return {"kind": kind, "tokens": _log(rng, 1, min(8192, most)), "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
                "rot": rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]), "interleaved": rng.random() < 0.4, "norm": rng.random() < 0.5,
                "layout": rng.choice(["apart", "packed", "gated"]), "base": rng.choice([1e4, 5e5, 1e6, 1e7]),
                "scaling": rng.choice(["none", "linear", "yarn"]), "far": rng.choice([0, 0, 30000, 900000]), "f32": f32}
    vocab = _log(rng, 1000, 250000)
    f32 = rng.random() < 0.5
    return {"kind": kind, "rows": _log(rng, 1, min(512, 421 * 248320 / (vocab * (2 if f32 else 1)))), "vocab": vocab, "pad": rng.choice([0, 0, rng.randint(1, 64)]),
            "top": rng.choice([0, 1, 5, 20, 32]), "temperature": rng.choice([1.0, 1.0, 0.8, 0.6, 1.5]), "masked": rng.choice([0.0, 0.0, 0.3, 0.9]), "f32": f32}


# ------------------------------------------------------------------ inputs

class Source:
    """Seeded tensors made on the GPU."""

    def __init__(self, seed: int):
        self.device = torch.device("cuda", torch.cuda.current_device())
        self.g = torch.Generator(device=self.device)
        self.g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 54321)

    def normal(self, *shape, scale: float = 1.0) -> torch.Tensor:
        return torch.randn(*shape, device=self.device, generator=self.g) * scale

    def uniform(self, *shape) -> torch.Tensor:
        return torch.rand(*shape, device=self.device, generator=self.g)

    def whole(self, most: int, *shape) -> torch.Tensor:
        return torch.randint(0, most, shape, device=self.device, generator=self.g)


def prepare(case: dict, seed: int) -> dict:
    s = Source(seed)
    make = {"route": _prepare_route, "rope": _prepare_rope, "logprobs": _prepare_logprobs}[case["kind"]]
    return {"case": case, **make(case, s)}


def run(state: dict):
    kind = state["case"]["kind"]
    if own:
        return {"route": _own_route, "rope": _own_rope, "logprobs": _own_logprobs}[kind](state)
    return {"route": _plain_route, "rope": _plain_rope, "logprobs": _plain_logprobs}[kind](state)


# ------------------------------------------------------------------ routing

def _prepare_route(c, s):
    """Router logits with experts of uneven popularity, and the small bias that evens them out."""
    t, e = c["tokens"], c["experts"]
    popular = s.normal(e, scale=0.5)
    logits = s.normal(t, e) + popular
    return {"logits": logits if c["f32"] else logits.half(),
            "bias": (-0.2 * popular + s.normal(e, scale=0.02)).contiguous() if c["bias"] else None,
            "idx": torch.empty((t, c["top_k"]), dtype=torch.int32, device=s.device), "w": torch.empty((t, c["top_k"]), dtype=torch.float32, device=s.device)}


def _own_route(st):
    from berth_b200 import moe
    c = st["case"]
    moe.route(st["logits"], st["bias"], st["idx"], st["w"], c["top_k"], score=c["score"], n_group=c["groups"], topk_group=c["keep"],
              group_score=c["group_score"], renormalize=c["renormalize"], scale=c["scale"])
    return {"idx": st["idx"], "w": st["w"]}


def _plain_route(st):
    """Scores in 64 bits: two experts' choice scores can lie closer than 32 bits tell apart."""
    c = st["case"]
    l = st["logits"].double()
    t, e = l.shape
    if c["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-l))
    else:
        ex = torch.exp(l - l.amax(1, keepdim=True))
        score = ex / ex.sum(1, keepdim=True)
    choice = score if st["bias"] is None else score + st["bias"].double()
    if c["groups"] > 1:
        ranked = torch.sort(choice.view(t, c["groups"], -1), dim=2, descending=True)[0]
        of_group = ranked[:, :, 0] if c["group_score"] == "max" else ranked[:, :, 0] + ranked[:, :, 1]
        kept = torch.sort(of_group, dim=1, descending=True, stable=True)[1][:, :c["keep"]]
        open_ = torch.zeros((t, c["groups"]), dtype=torch.bool, device=l.device).scatter_(1, kept, True)
        choice = torch.where(open_.repeat_interleave(e // c["groups"], 1), choice, -math.inf)
    idx = torch.sort(choice, dim=1, descending=True, stable=True)[1][:, :c["top_k"]]
    w = score.gather(1, idx)
    if c["renormalize"]:
        w = w / w.sum(1, keepdim=True)
    return {"idx": idx.int(), "w": (w * c["scale"]).float()}


def _exact_route(c, st):
    """The weights from differences of logits: a softmax is 1 / sum of exp(l_j - l_i), a sigmoid a half of 1 + tanh(l / 2)."""
    l = st["logits"].double()
    t, e = l.shape
    if c["score"] == "sigmoid":
        score = 0.5 * (1.0 + torch.tanh(0.5 * l))
        score = torch.where(l < -8, torch.exp(l - torch.log1p(torch.exp(l))), score)
    else:
        score = torch.exp(torch.log_softmax(l, 1))
    choice = score if st["bias"] is None else score + st["bias"].double()
    if c["groups"] > 1:
        g = choice.view(t, c["groups"], -1)
        best = g.topk(1 if c["group_score"] == "max" else 2, dim=2)[0].sum(2)
        # a group stays if fewer than `keep` come before it
        before = (best[:, None, :] > best[:, :, None]) | ((best[:, None, :] == best[:, :, None]) & _lower(c["groups"], l.device))
        choice = g.masked_fill((before.sum(2) >= c["keep"])[:, :, None], -math.inf).view(t, e)
    idx = torch.argsort(-choice, dim=1, stable=True)[:, :c["top_k"]]
    w = score.gather(1, idx)
    return {"idx": None, "w": c["scale"] * (w / w.sum(1, keepdim=True) if c["renormalize"] else w)}


def _lower(n, device):
    i = torch.arange(n, device=device)
    return i[None, :] < i[:, None]


# ------------------------------------------------------------------ rotary positions

EPS, NORM_BIAS = 1e-6, 1.0      # the norms' weights are stored around zero


def _frequencies(c):
    """Radians per position of each pair, and the factor on cos and sin: plain, divided by the stretch, or blended between the
    two by how often a pair turns within the context that was trained (32 turns and more: plain, one or less: divided)."""
    half = c["rot"] // 2
    f = [c["base"] ** (-2.0 * i / c["rot"]) for i in range(half)]
    if c["scaling"] == "linear":
        return [v / 8.0 for v in f], 1.0
    if c["scaling"] == "yarn":
        at = [c["rot"] * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(c["base"])) for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), c["rot"] - 1)
        ramp = [min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for i in range(half)]
        return [v * (1 - r) + v / 32.0 * r for v, r in zip(f, ramp)], 0.1 * math.log(32.0) + 1.0
    return f, 1.0


def _prepare_rope(c, s):
    """q and k as the projections leave them: apart, as columns of one q/k/v buffer, or q with a gate behind each head."""
    t, hq, hk, d = c["tokens"], c["q_heads"], c["k_heads"], c["dim"]
    dt = torch.float32 if c["f32"] else torch.float16
    if c["layout"] == "packed":
        qkv = s.normal(t, hq + 2 * hk, d).to(dt)
        q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    else:
        q = s.normal(t, hq, 2 * d if c["layout"] == "gated" else d).to(dt)[:, :, :d]
        k = s.normal(t, hk, d).to(dt)
    # chunks of up to three sequences, each at a place of its own
    cut = torch.sort(s.whole(t, 2))[0]
    i = torch.arange(t, device=s.device)
    begin = s.whole(4096, 3) + c["far"]
    position = i + torch.where(i < cut[0], begin[0], torch.where(i < cut[1], begin[1] - cut[0], begin[2] - cut[1]))
    f, factor = _frequencies(c)
    norm = lambda: s.normal(d, scale=0.05).bfloat16() if c["norm"] else None
    return {"q": q, "k": k, "position": position.int(), "inv_freq": torch.tensor(f, dtype=torch.float64, device=s.device), "factor": factor,
            "q_norm": norm(), "k_norm": norm(), "q_out": torch.empty((t, hq, d), dtype=dt, device=s.device),
            "k_out": torch.empty((t, hk, d), dtype=dt, device=s.device)}


def _own_rope(st):
    from berth_b200.kernels import ops
    c = st["case"]
    ops.rope(st["q"], st["k"], st["position"], st["inv_freq"], st["q_out"], st["k_out"], c["interleaved"], st["factor"], st["q_norm"], st["k_norm"],
             EPS, NORM_BIAS)
    return {"q": st["q_out"], "k": st["k_out"]}


def _plain_rope(st):
    c = st["case"]
    angle = st["position"].double()[:, None, None] * st["inv_freq"]      # far positions turn through more angle than 32 bits hold
    cos, sin = ((st["factor"] * v).float() for v in (torch.cos(angle), torch.sin(angle)))
    return {"q": _plain_turn(c, st["q"], st["q_norm"], cos, sin), "k": _plain_turn(c, st["k"], st["k_norm"], cos, sin)}


def _plain_turn(c, x, norm, cos, sin):
    y = x.float()
    if norm is not None:
        y = y * torch.rsqrt((y * y).mean(2, keepdim=True) + EPS) * (norm.float() + NORM_BIAS)
    r = c["rot"]
    a, b = (y[:, :, 0:r:2], y[:, :, 1:r:2]) if c["interleaved"] else (y[:, :, :r // 2], y[:, :, r // 2:r])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), 3).flatten(2) if c["interleaved"] else torch.cat((a, b), 2)
    return torch.cat((turned, y[:, :, r:]), 2).to(x.dtype)


def _exact_rope(c, st):
    """Pairs as complex numbers times factor * exp(i * angle)."""
    turn = torch.polar(torch.full((c["tokens"], c["rot"] // 2), st["factor"], dtype=torch.float64, device=st["q"].device),
                       st["position"].double()[:, None] * st["inv_freq"][None, :])[:, None, :]
    out = {}
    for name in ("q", "k"):
        y = st[name].double()
        if c["norm"]:
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * (st[name + "_norm"].double() + NORM_BIAS)
        head = y[..., :c["rot"]]
        pairs = head.unflatten(-1, (-1, 2)) if c["interleaved"] else head.unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        out[name] = torch.cat(((z if c["interleaved"] else z.transpose(-1, -2)).flatten(-2), y[..., c["rot"]:]), -1)
    return out


# ------------------------------------------------------------------ log probabilities

def _prepare_logprobs(c, s):
    """Logits of rows between undecided and certain; the token is mostly a likely one; a grammar's mask is -inf."""
    r, v = c["rows"], c["vocab"]
    logits = s.normal(r, v + c["pad"], scale=2.5)
    likely = s.whole(v, r, 8)
    logits.scatter_add_(1, likely, s.uniform(r, 8) * 16.0)
    if c["masked"]:
        logits.masked_fill_(s.uniform(r, v + c["pad"]) < c["masked"], -math.inf)
        logits.scatter_(1, likely[:, :2], 9.0)        # the grammar always leaves something
    token = torch.where(s.uniform(r) < 0.75, likely[:, 0], s.whole(v, r))
    f32, i32 = (dict(dtype=dt, device=s.device) for dt in (torch.float32, torch.int32))
    return {"logits": logits if c["f32"] else logits.half(), "token": token.int(), "logprob": torch.empty(r, **f32), "rank": torch.empty(r, **i32),
            "entropy": torch.empty(r, **f32), "top": torch.empty((r, c["top"]), **i32), "top_logprob": torch.empty((r, c["top"]), **f32)}


def _own_logprobs(st):
    from berth_b200.kernels import ops
    c = st["case"]
    ops.logprobs(st["logits"], st["token"], st["logprob"], st["rank"], st["entropy"], st["top"], st["top_logprob"], c["vocab"], 1.0 / c["temperature"])
    return {k: st[k] for k in ("logprob", "rank", "entropy", "top", "top_logprob")}


def _plain_logprobs(st):
    c = st["case"]
    x = st["logits"][:, :c["vocab"]]
    token = st["token"].long()[:, None]
    # the order of the vocabulary, whole numbers: the larger logit first, then the lower token
    bits = (x.float() + 0.0).view(torch.int32).long()
    order = (torch.where(bits < 0, -(bits & 0x7fffffff), bits) << 20) + (1048575 - torch.arange(c["vocab"], device=x.device))
    rank = (order > order.gather(1, token)).sum(1)
    top = 1048575 - (torch.topk(order, c["top"], 1)[0] & 1048575) if c["top"] else order[:, :0]
    z = x.float() / c["temperature"]
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    entropy = lse - torch.where(e > 0, e * z, 0.0).sum(1, keepdim=True) / total
    return {"logprob": (z.gather(1, token) - lse)[:, 0], "rank": rank.int(), "entropy": entropy[:, 0], "top": top.int(), "top_logprob": z.gather(1, top) - lse}


def _exact_logprobs(c, st):
    z = st["logits"][:, :c["vocab"]].double() / c["temperature"]
    lp = z - torch.logsumexp(z, 1, keepdim=True)
    entropy = -(lp.exp() * lp.clamp(min=-1e4)).sum(1)
    best = torch.sort(lp, 1, descending=True)[0][:, :c["top"]] if c["top"] else lp[:, :0]
    return {"logprob": lp.gather(1, st["token"].long()[:, None])[:, 0], "rank": None, "entropy": entropy, "top": None, "top_logprob": best}


# ------------------------------------------------------------------ from the definition, and the work of a pass

def exact(case: dict, seed: int):
    st = prepare(case, seed)
    return {"route": _exact_route, "rope": _exact_rope, "logprobs": _exact_logprobs}[case["kind"]](case, st)


def work(case: dict) -> dict:
    c = case
    size = 4 if c["f32"] else 2
    if c["kind"] == "route":        # a score per expert, an add and a comparison
        n = c["tokens"] * c["experts"]
        return {"bytes": n * size + (4 * c["experts"] if c["bias"] else 0) + 8 * c["tokens"] * c["top_k"], "flops": 6.0 * n}
    if c["kind"] == "rope":         # every element of q and k in and out; a pair's two products of two, four operations an element of a norm
        heads = c["tokens"] * (c["q_heads"] + c["k_heads"])
        return {"bytes": 2 * heads * c["dim"] * size + 4 * c["tokens"] + 4 * c["rot"] + (4 * c["dim"] if c["norm"] else 0),
                "flops": heads * (3.0 * c["rot"] + (4.0 * c["dim"] if c["norm"] else 0))}
    n = c["rows"] * c["vocab"]      # scale, exp, its sum, the entropy's product and sum, two comparisons
    return {"bytes": n * size + c["rows"] * (16 + 8 * c["top"]), "flops": 7.0 * n}

"""Performance cases of the policy's operators: the memory that a policy keeps over its observations.

A trainer that steps up to 1024 environments feeds each frame's features to a policy with a
memory, reads it once a step while acting and again over whole rollouts while learning. The
operators are the gated delta rule in its two forms (``gated_delta_step`` for one token of
every environment, ``gated_delta_rule`` for rollouts, with gradients), the pass that
prepares its queries and keys (``qk_norm``) and the clipping of the update
(``clip_grad_norm``). Batches are those of the benchmark and of ``bench_sdfdag`` (1 to 1024
environments, 128 steps), heads and lengths generic, odd sizes beside them.

Per value head, with a state S of K x V numbers and a = 0 at an episode's first token, exp(g)
elsewhere: u = v - a S'k, S <- a S + beta k u', o = scale S'q.
"""

from __future__ import annotations

import math

import torch

DEVICE = "cuda"
CHUNK = 64  # tokens that the plain form takes at once
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}

own = False


def listed():
    return [
        # one actor thinks for one frame: the latency of a single call
        _step("step_one_actor", 1, 4, 8, 128, 128, "bfloat16", starts=False),
        # bench_sdfdag's default count of actors, heads of a small policy, episodes that begin
        _step("step_64_actors", 64, 4, 4, 64, 64, "float32"),
        # the benchmark's full batch of environments: 268 MB of states, read and written
        _step("step_1024_envs", 1024, 4, 4, 128, 128, "bfloat16"),
        # an evaluation pass over a short rollout, with the state carried in and out
        _rule("rollout_64_actors", 64, 128, 4, 4, 64, 64, "float16", state=True),
        # a long recorded walk replayed through the memory: few heads, a long chain
        _rule("long_walk", 1, 16384, 8, 16, 128, 128, "bfloat16", starts=False, state=True),
        # a small learner in 32 bits, sizes that divide by nothing, truncated in time
        _rule("learn_odd_f32", 9, 77, 2, 6, 48, 80, "float32", grad=True, state=True),
        # a long sequence of which two key heads serve four value heads each
        _rule("learn_long", 2, 4001, 2, 8, 128, 128, "bfloat16", grad=True),
        # the learner's minibatch: every environment of the benchmark, 128 steps
        _rule("learn_1024_envs", 1024, 128, 4, 4, 64, 64, "bfloat16", grad=True),
        # queries and keys of one frame of 64 actors: launch latency
        _norm("norm_64_actors", 64, 1, 4, 4, 64, 64, "l2", "float32"),
        # the learner's pass over the same minibatch, learned scales, their gradients
        _norm("norm_learn", 1024, 128, 4, 4, 64, 32, "rms", "bfloat16", weights=True, grad=True),
        # the update of a small policy in 32 bits
        _clip("clip_policy", 4, 256, "float32"),
        # the update of a large one, master gradients in 32 bits
        _clip("clip_large", 24, 2000, "float32"),
    ]


def draw(rng):
    kind = rng.choice(["step", "rule", "learn", "rule", "learn", "norm", "norm", "clip"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    starts = rng.random() < 0.6
    hk = rng.choice([1, 2, 3, 4, 8])
    hv = hk * rng.choice([1, 1, 2, 3, 4])
    if kind == "clip":
        return _clip(None, rng.randint(1, 24), _spread(rng, 24, 2000), dtype, max_norm=rng.choice([0.5, 1.0, 1.0, 1e4]))
    if kind == "norm":
        d = rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 256])
        grad = rng.random() < 0.5
        t = _spread(rng, 1, 2048)
        b = _spread(rng, 1, max(1, min(1024, (1 << 26) // (t * (hk + hv) * d))))
        return _norm(None, b, t, hv, hk, d, rng.choice([0, d, d // 2]), rng.choice(["l2", "rms"]), dtype,
                     weights=rng.random() < 0.6, grad=grad, interleaved=rng.random() < 0.3)
    k, v = (rng.choice([16, 24, 32, 48, 64, 64, 64, 80, 96, 128, 128, rng.randint(9, 127)]) for _ in range(2))
    if kind == "step":
        b = _spread(rng, 1, max(1, min(1024, (1 << 26) // (hv * k * v))))
        return _step(None, b, hk, hv, k, v, dtype, starts=starts)
    grad = kind == "learn"
    t = _spread(rng, 1, 4096 if grad else 16384)
    most = min((1 << (31 if grad else 32)) // (t * hv * k * v), (1 << 26) // (t * hv * (k + v)),
               (1 << 26) // (hv * k * v))
    b = _spread(rng, 1, max(1, min(1024, most)))
    return _rule(None, b, t, hk, hv, k, v, dtype, starts=starts, state=rng.random() < 0.5, grad=grad)


def _named(name, case):
    return case if name is None else {"name": name, **case}


def _step(name, envs, hk, hv, k, v, dtype, starts=True):
    return _named(name, {"op": "step", "envs": envs, "key_heads": hk, "value_heads": hv, "key_dim": k,
                         "value_dim": v, "dtype": dtype, "starts": starts})


def _rule(name, envs, steps, hk, hv, k, v, dtype, starts=True, state=False, grad=False):
    return _named(name, {"op": "rule", "envs": envs, "steps": steps, "key_heads": hk, "value_heads": hv,
                         "key_dim": k, "value_dim": v, "dtype": dtype, "starts": starts, "state": state,
                         "grad": grad})


def _norm(name, envs, steps, hq, hk, dim, rotary, kind, dtype, weights=False, grad=False, interleaved=False):
    return _named(name, {"op": "norm", "envs": envs, "steps": steps, "query_heads": hq, "key_heads": hk, "dim": dim,
                         "rotary": rotary, "norm": kind, "dtype": dtype, "weights": weights, "grad": grad,
                         "interleaved": interleaved})


def _clip(name, layers, width, dtype, max_norm=1.0):
    return _named(name, {"op": "clip", "layers": layers, "width": width, "dtype": dtype, "max_norm": max_norm})


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = min(hi, max(lo, n))
    return n - 1 if n == 3072 else n


def _clip_shapes(case):
    """The parameters of a policy of ``layers`` blocks: an encoder's first product of odd
    size, four square products, one to twice the width and one back, scales, a head of seven actions."""
    w = case["width"]
    block = [(w, w)] * 4 + [(2 * w, w), (w, 2 * w), (w,), (w,)]
    return [(w, 105)] + block * case["layers"] + [(7, w), (7,), (1,)]


# ---- what a user's program has in hand ----


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return {"case": case, **_PREPARE[case["op"]](case, gen)}


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE)


def _memory_inputs(case, gen, lead):
    """Features that change slowly from frame to frame, so that keys are alike (unit norm), gates
    of a sigmoid, decays from nearly none to a factor of three a step, and episodes that end."""
    hk, hv, k, v = case["key_heads"], case["value_heads"], case["key_dim"], case["value_dim"]
    dtype = TYPES[case["dtype"]]
    common = _randn(gen, lead[0], *([1] * (len(lead) - 1)), hk, k)
    s = {
        "q": torch.nn.functional.normalize(_randn(gen, *lead, hk, k), dim=-1).to(dtype),
        "k": torch.nn.functional.normalize(_randn(gen, *lead, hk, k) + 0.6 * common, dim=-1).to(dtype),
        "v": _randn(gen, *lead, hv, v).to(dtype),
        "g": -torch.exp(_randn(gen, *lead, hv) * 1.5 - 3.0).clamp(max=1.2),
        "beta": torch.sigmoid(_randn(gen, *lead, hv) + 0.5),
        "starts": torch.rand(lead, generator=gen, device=DEVICE) < 1.0 / 50 if case["starts"] else None,
    }
    if case["op"] == "step" or case["state"]:
        s["state"] = 0.3 * _randn(gen, lead[0], hv, k, v)
    return s


def _prepare_step(case, gen):
    return _memory_inputs(case, gen, (case["envs"],))


def _prepare_rule(case, gen):
    s = _memory_inputs(case, gen, (case["envs"], case["steps"]))
    if case["grad"]:
        s["grad_o"] = _randn(gen, *s["v"].shape).to(s["v"].dtype)
        if case["state"]:
            s["grad_state"] = 0.3 * _randn(gen, *s["state"].shape)
        for x in ("q", "k", "v", "g", "beta", "state"):
            if x in s:
                s[x].requires_grad_()
    return s


def _prepare_norm(case, gen):
    b, t, d, r = case["envs"], case["steps"], case["dim"], case["rotary"]
    dtype = TYPES[case["dtype"]]
    s = {x: (_randn(gen, b, t, case[h], d) * torch.exp(0.5 * _randn(gen, b, t, 1, 1))).to(dtype)
         for x, h in (("q", "query_heads"), ("k", "key_heads"))}
    if case["weights"]:
        s["q_weight"], s["k_weight"] = (1.0 + 0.2 * _randn(gen, d) for _ in range(2))
    if r:
        # a step's place in its episode: environments are anywhere in theirs when a rollout begins
        first = torch.randint(0, 512, (b, 1), generator=gen, device=DEVICE)
        s["positions"] = (first + torch.arange(t, device=DEVICE)).to(torch.int32)
        angle = torch.arange(512 + t, device=DEVICE)[:, None] * 10000.0 ** (
            -torch.arange(r // 2, device=DEVICE) / max(1, r // 2))
        s["cos"], s["sin"] = torch.cos(angle), torch.sin(angle)
    if case["grad"]:
        s["grad_q"], s["grad_k"] = (_randn(gen, *s[x].shape).to(dtype) for x in ("q", "k"))
        for x in ("q", "k", "q_weight", "k_weight"):
            if x in s:
                s[x].requires_grad_()
    return s


def _prepare_clip(case, gen):
    dtype = TYPES[case["dtype"]]
    shapes = _clip_shapes(case)
    sizes = [math.prod(x) for x in shapes]
    level = 6.0 / math.sqrt(sum(sizes))  # a norm of a few times the limit
    grads = [(level * math.exp(0.6 * ((7 * i) % 5 - 2)) * _randn(gen, *x)).to(dtype) for i, x in enumerate(shapes)]
    flat = torch.empty(sum(sizes), dtype=dtype, device=DEVICE)  # what the optimizer reads
    out = [x.view(y) for x, y in zip(flat.split(sizes), shapes)]
    return {"grads": grads, "flat": flat, "out": out}


_PREPARE = {"step": _prepare_step, "rule": _prepare_rule, "norm": _prepare_norm, "clip": _prepare_clip}


# ---- one pass ----


def run(state):
    op = state["case"]["op"]
    return _OWN[op](state) if own else _PLAIN[op](state)


def _own_step(s):
    from navi_amd import policy

    o = policy.gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], starts=s["starts"])
    return {"o": o, "state": s["state"]}


def _own_rule(s):
    from navi_amd import policy

    carried = s["case"]["state"]
    got = policy.gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], starts=s["starts"],
                                  initial_state=s.get("state"), return_state=carried)
    o, final = got if carried else (got, None)
    return _with_gradients(s, {"o": o, "state": final} if carried else {"o": o},
                           [o, final] if carried else [o], ["grad_o", "grad_state"],
                           ["q", "k", "v", "g", "beta", "state"])


def _own_norm(s):
    from navi_amd import policy

    c = s["case"]
    q, k = policy.qk_norm(s["q"], s["k"], q_weight=s.get("q_weight"), k_weight=s.get("k_weight"), norm=c["norm"],
                          cos=s.get("cos"), sin=s.get("sin"), positions=s.get("positions"),
                          interleaved=c["interleaved"])
    return _with_gradients(s, {"q": q, "k": k}, [q, k], ["grad_q", "grad_k"], ["q", "k", "q_weight", "k_weight"])


def _own_clip(s):
    from navi_amd import policy

    norm = policy.clip_grad_norm(s["grads"], s["case"]["max_norm"], out=s["out"])
    return {"norm": norm, "clipped": s["flat"]}


_OWN = {"step": _own_step, "rule": _own_rule, "norm": _own_norm, "clip": _own_clip}


def _with_gradients(s, outputs, of, given, inputs):
    """The outputs, in a learner's pass with the gradients of the inputs beside them."""
    if not s["case"]["grad"]:
        return outputs
    wanted = [x for x in inputs if x in s]
    grads = torch.autograd.grad(of, [s[x] for x in wanted], [s[x] for x in given[:len(of)]])
    return {**{x: y.detach() for x, y in outputs.items()}, **{"d_" + x: y for x, y in zip(wanted, grads)}}


# ---- the plain forms, in 32 bits ----


def _per_value_head(x, heads, axis):
    return x.float().repeat_interleave(heads // x.shape[axis], dim=axis)


def _plain_step(s):
    hv = s["case"]["value_heads"]
    q, k = (_per_value_head(s[x], hv, 1) for x in ("q", "k"))
    a = torch.exp(s["g"])
    if s["starts"] is not None:
        a = torch.where(s["starts"][:, None], torch.zeros_like(a), a)
    state = a[..., None, None] * s["state"]
    u = s["v"].float() - (k[..., None] * state).sum(-2)
    state = state + (s["beta"][..., None] * k)[..., None] * u[..., None, :]
    o = s["case"]["key_dim"] ** -0.5 * (q[..., None] * state).sum(-2)
    s["state"].copy_(state)
    return {"o": o.to(s["v"].dtype), "state": s["state"]}


def _plain_rule(s):
    c = s["case"]
    b, t, hv = c["envs"], c["steps"], c["value_heads"]
    n = -(-t // CHUNK)
    pad = n * CHUNK - t

    def chunks(x):  # [B, T, H, ...] -> [B, H, N, CHUNK, ...], zeros after the last token
        x = torch.cat([x, x.new_zeros(b, pad, *x.shape[2:])], 1) if pad else x
        return x.transpose(1, 2).reshape(b, x.shape[2], n, CHUNK, *x.shape[3:])

    q, k = (chunks(_per_value_head(s[x], hv, 2)) for x in ("q", "k"))
    v, beta, g = chunks(s["v"].float()), chunks(s["beta"]), chunks(s["g"])
    first = torch.zeros_like(g, dtype=torch.bool)
    if s["starts"] is not None:
        first = chunks(s["starts"][..., None].expand(b, t, hv))
    total = torch.cumsum(torch.where(first, torch.zeros_like(g), g), -1)
    episode = torch.cumsum(first.int(), -1)
    row = torch.arange(CHUNK, device=g.device)
    within = (episode[..., :, None] == episode[..., None, :]) & (row[:, None] >= row)
    decay = torch.exp((total[..., :, None] - total[..., None, :]).masked_fill(~within, -math.inf))
    from_first = torch.exp(total.masked_fill(episode != 0, -math.inf))
    to_last = torch.exp((total[..., -1:] - total).masked_fill(episode != episode[..., -1:], -math.inf))
    inverse = _unit_lower_inverse((beta[..., None] * decay * (k @ k.transpose(-1, -2))).tril(-1))
    values = inverse @ (beta[..., None] * v)
    keys = inverse @ ((beta * from_first)[..., None] * k)
    scale = c["key_dim"] ** -0.5
    weights = scale * decay * (q @ k.transpose(-1, -2))
    queries = (scale * from_first)[..., None] * q
    left = (to_last[..., None] * k).transpose(-1, -2)
    keep = from_first[..., -1, None, None]
    state = s["state"] if "state" in s else k.new_zeros(b, hv, c["key_dim"], c["value_dim"])
    out = []
    for i in range(n):  # a chunk needs the state that the one before it leaves
        w = values[:, :, i] - keys[:, :, i] @ state
        out.append(queries[:, :, i] @ state + weights[:, :, i] @ w)
        state = keep[:, :, i] * state + left[:, :, i] @ w
    o = torch.stack(out, 2).reshape(b, hv, n * CHUNK, -1)[:, :, :t].transpose(1, 2).to(s["v"].dtype)
    carried = c["state"]
    return _with_gradients(s, {"o": o, "state": state} if carried else {"o": o}, [o, state] if carried else [o],
                           ["grad_o", "grad_state"], ["q", "k", "v", "g", "beta", "state"])


def _unit_lower_inverse(a):
    """(I + a)^-1 of strictly lower triangles, from the inverses of diagonal blocks of 1, 2, 4, ...:
    the block below two of them is -(the lower's) a (the upper's)."""
    row = torch.arange(a.shape[-1], device=a.device)
    inverse = torch.eye(a.shape[-1], device=a.device).expand_as(a)
    size = 1
    while size < a.shape[-1]:
        pair = (row[:, None] // (2 * size) == row // (2 * size)) & (row[:, None] // size != row // size)
        inverse = inverse - inverse @ (a * pair) @ inverse
        size *= 2
    return inverse


def _plain_norm(s):
    c = s["case"]
    got = {}
    for x in ("q", "k"):
        y = s[x].float()
        square = y.square().sum(-1, keepdim=True)
        y = y * torch.rsqrt((square / c["dim"] if c["norm"] == "rms" else square) + 1e-6)
        y = y * s[x + "_weight"] if c["weights"] else y
        got[x] = (_turned(y, s, c) if c["rotary"] else y).to(s[x].dtype)
    return _with_gradients(s, got, [got["q"], got["k"]], ["grad_q", "grad_k"], ["q", "k", "q_weight", "k_weight"])


def _turned(y, s, c):
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    r = c["rotary"]
    if c["interleaved"]:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), y[..., r:]], -1)
    a, b = y[..., :r // 2], y[..., r // 2:r]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., r:]], -1)


def _plain_clip(s):
    norm = torch.sqrt(torch.stack([x.float().square().sum() for x in s["grads"]]).sum())
    factor = torch.clamp(s["case"]["max_norm"] / (norm + 1e-6), max=1.0)
    clipped = torch.cat([(x.float() * factor).to(x.dtype).reshape(-1) for x in s["grads"]])
    return {"norm": norm, "clipped": clipped}


_PLAIN = {"step": _plain_step, "rule": _plain_rule, "norm": _plain_norm, "clip": _plain_clip}


# ---- what a pass cannot do without ----


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "clip":
        n = sum(math.prod(x) for x in _clip_shapes(case))
        return {"bytes": 2 * n * e + 4, "flops": 3 * n}
    b, t = case["envs"], case.get("steps", 1)
    if case["op"] == "norm":
        n = b * t * (case["query_heads"] + case["key_heads"]) * case["dim"]
        r = b * t * (case["query_heads"] + case["key_heads"]) * case["rotary"]
        tables = (b * t * 4 + (512 + t) * case["rotary"] * 4) if case["rotary"] else 0
        passes = 2 if not case["grad"] else 4  # gradients: theirs is read and that of the input written as well
        return {"bytes": passes * n * e + tables, "flops": (4 * n + 3 * r) * (3 if case["grad"] else 1)}
    hk, hv, k, v = case["key_heads"], case["value_heads"], case["key_dim"], case["value_dim"]
    inputs = b * t * (e * (2 * hk * k + hv * v) + 8 * hv + (1 if case["starts"] else 0))
    out = b * t * hv * v * e
    flops = 7 * b * t * hv * k * v  # S'k, the update and S'q of the recurrence
    states = 4 * b * hv * k * v
    if case["op"] == "step":
        return {"bytes": inputs + out + 2 * states, "flops": flops}
    total = inputs + out + (2 * states if case["state"] else 0)
    if case["grad"]:  # of the output in, those of the inputs out
        total += out + b * t * (e * (2 * hk * k + hv * v) + 8 * hv) + (2 * states if case["state"] else 0)
        flops *= 3
    return {"bytes": total, "flops": flops}


# ---- the definitions in 64 bits ----


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _EXACT[case["op"]](case, {x: y.double() if torch.is_tensor(y) and y.is_floating_point() else y
                                         for x, y in s.items() if x not in ("grads", "flat", "out")}, s)


def _exact_step(case, s, _given):
    o, state = _exact_token({**s, "S": s["state"]}, case, lambda x: x)[:2]
    return {"o": o, "state": state}


def _exact_token(s, case, of):
    """One token of the recurrence: (o, state after it, state before it, a, u, S'k)."""
    rep = case["value_heads"] // case["key_heads"]
    q, k = (of(s[x]).repeat_interleave(rep, 1) for x in ("q", "k"))
    a = torch.exp(of(s["g"]))
    if s["starts"] is not None:
        a = a * (~of(s["starts"]))[:, None]
    before = s["S"]
    read = torch.einsum("bhkv,bhk->bhv", before, k)
    u = of(s["v"]) - a[..., None] * read
    state = a[..., None, None] * before + torch.einsum("bhk,bhv->bhkv", of(s["beta"])[..., None] * k, u)
    o = torch.einsum("bhkv,bhk->bhv", state, q) * case["key_dim"] ** -0.5
    return o, state, before, a, u, read


def _exact_rule(case, s, _given):
    b, t, hk, hv, kd, vd = (case[x] for x in ("envs", "steps", "key_heads", "value_heads", "key_dim", "value_dim"))
    if case["grad"] and 8 * b * t * hv * kd * vd > 70e9:
        return None  # a state for every token does not fit
    rep = hv // hk
    start = s["state"] if "state" in s else torch.zeros(b, hv, kd, vd, dtype=torch.float64, device=DEVICE)
    s = {**s, "S": start}
    o = torch.empty(b, t, hv, vd, dtype=torch.float64, device=DEVICE)
    tape = []
    for i in range(t):
        o[:, i], s["S"], *rest = _exact_token(s, case, lambda x: x[:, i])
        if case["grad"]:
            tape.append(rest)
    got = {"o": o, **({"state": s["S"]} if case["state"] else {})}
    if not case["grad"]:
        return got
    d = {x: torch.empty_like(s[x]) for x in ("q", "k", "v", "g", "beta")}
    ds = s["grad_state"].clone() if case["state"] else torch.zeros_like(start)
    after = s["S"]
    for i in reversed(range(t)):
        before, a, u, read = tape.pop()
        q, k = (s[x][:, i].repeat_interleave(rep, 1) for x in ("q", "k"))
        do, beta = s["grad_o"][:, i] * kd ** -0.5, s["beta"][:, i]
        ds = ds + torch.einsum("bhk,bhv->bhkv", q, do)
        dq = torch.einsum("bhkv,bhv->bhk", after, do)
        dsu = torch.einsum("bhkv,bhv->bhk", ds, u)
        du = beta[..., None] * torch.einsum("bhkv,bhk->bhv", ds, k)
        dk = beta[..., None] * dsu - a[..., None] * torch.einsum("bhkv,bhv->bhk", before, du)
        da = (before * ds).sum((-1, -2)) - (du * read).sum(-1)
        d["q"][:, i], d["k"][:, i] = (x.view(b, hk, rep, kd).sum(2) for x in (dq, dk))
        d["v"][:, i], d["beta"][:, i], d["g"][:, i] = du, (k * dsu).sum(-1), a * da
        ds = a[..., None, None] * (ds - torch.einsum("bhk,bhv->bhkv", k, du))
        after = before
    got.update({"d_" + x: y for x, y in d.items()})
    return {**got, "d_state": ds} if case["state"] else got


def _exact_norm(case, s, _given):
    got, grads = {}, {}
    for x in ("q", "k"):
        y, w = s[x], s.get(x + "_weight", torch.ones(case["dim"], dtype=torch.float64, device=DEVICE))
        count = case["dim"] if case["norm"] == "rms" else 1
        inv = 1.0 / torch.sqrt((y * y).sum(-1, keepdim=True) / count + 1e-6)
        got[x] = _exact_turn(y * inv * w, s, case, 1.0)
        if case["grad"]:
            dz = _exact_turn(s["grad_" + x], s, case, -1.0)
            dn = dz * w
            grads["d_" + x] = inv * dn - y * inv ** 3 * (dn * y).sum(-1, keepdim=True) / count
            if case["weights"]:
                grads["d_" + x + "_weight"] = (dz * y * inv).sum((0, 1, 2))
    return {**got, **grads}


def _exact_turn(y, s, case, way):
    r = case["rotary"]
    if not r:
        return y
    at = s["positions"].long()
    turn = torch.complex(s["cos"][at], way * s["sin"][at])[:, :, None]
    if case["interleaved"]:
        z = torch.view_as_complex(y[..., :r].unflatten(-1, (r // 2, 2)).contiguous()) * turn
        head = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(y[..., :r // 2].contiguous(), y[..., r // 2:r].contiguous()) * turn
        head = torch.cat([z.real, z.imag], -1)
    return torch.cat([head, y[..., r:]], -1)


def _exact_clip(case, _s, given):
    flat = torch.cat([x.reshape(-1) for x in given["grads"]]).double()
    norm = torch.linalg.vector_norm(flat)
    return {"norm": norm, "clipped": flat * min(1.0, case["max_norm"] / (float(norm) + 1e-6))}


_EXACT = {"step": _exact_step, "rule": _exact_rule, "norm": _exact_norm, "clip": _exact_clip}

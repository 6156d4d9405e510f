"""Performance cases of a policy's selective memory: the block around it, and its update.

Another temporal core over the tracer's observations than the gated delta rule's: a short
convolution of the last frames (``causal_conv``, ``causal_conv_step``), a selective state space
scan (``selective_scan`` over rollouts, with gradients, ``selective_scan_step`` for one frame),
the norms, gate and residual sum around such a block (``block_norm``), and the update of its
matrices by Newton-Schulz products (``orthogonalize``). Batches are those of the benchmark and
of ``bench_sdfdag`` (1 to 1024 environments, 128 steps), widths those of ``memory_policy`` and
generic ones, odd sizes beside them.

Convolution, per channel: z[t] = bias + sum_j weight[j] x[t - (taps - 1) + j], y = silu(z), where
inputs of another episode count as 0. Scan, per head, with a state S of N x P numbers:
beta = softplus(dt + dt_bias), S <- exp(beta a) S + beta B x' (S = 0 before an episode's first
token), y = S'C + d x. Block: m = norm(y) post silu(gate), h = residual + scale m, and
norm(h) pre, with norm(x) = x / sqrt(mean x^2 + eps). Update: X = G / (|G| + eps), then five times
X <- 3.4445 X - 4.775 A X + 2.0315 A A X with A = X X' (X the wide one of G and its transpose).
"""

from __future__ import annotations

import math

import torch

DEVICE = "cuda"
CHUNK = 64  # tokens that the plain scan takes at once
EPS = 1e-6
STEPS = 5
FACTORS = (3.4445, -4.775, 2.0315)
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
BYTES = {"bfloat16": 2, "float16": 2, "float32": 4}

own = False


def listed():
    return [
        # one actor thinks for one frame: the latency of a single call
        _step("scan_step_one_actor", 1, 8, 1, 128, 64, "bfloat16", starts=False),
        # the benchmark's full batch of environments: 268 MB of states, read and written
        _step("scan_step_1024_envs", 1024, 8, 2, 128, 64, "bfloat16"),
        # an evaluation pass of bench_sdfdag's actors over a short rollout, the state carried in and out
        _scan("scan_rollout_64_actors", 64, 128, 4, 4, 64, 64, "float16", state=True),
        # a long recorded walk replayed through the memory: a long chain, one group of B and C
        _scan("scan_long_walk", 1, 16384, 16, 1, 128, 64, "bfloat16", starts=False, state=True),
        # a small learner in 32 bits, sizes that divide by nothing, truncated in time
        _scan("scan_learn_odd_f32", 9, 77, 6, 2, 48, 80, "float32", grad=True, state=True),
        # the learner's minibatch: every environment of the benchmark, 128 steps
        _scan("scan_learn_1024_envs", 1024, 128, 4, 1, 64, 64, "bfloat16", grad=True),
        # the convolution of one frame of 64 actors: launch latency
        _conv("conv_step_64_actors", 64, 0, 384, 4, "float32"),
        # the learner's pass over the same minibatch: x, B and C of four heads of 64, one group
        _conv("conv_learn_1024_envs", 1024, 128, 384, 4, "bfloat16", grad=True),
        # one frame of 64 actors through the end of a block of memory_policy's width
        _block("block_64_actors", 64, 1, 256, "float32"),
        # the learner's pass, a residual stream in 32 bits, every gradient
        _block("block_learn_1024_envs", 1024, 128, 256, "bfloat16", wide_residual=True, grad=True),
        # the update of a small policy, in 32 bits
        _update("update_policy", 4, 256, "float32", "float32"),
        # the update of a large one for weights in 16 bits
        _update("update_large", 8, 2000, "float32", "bfloat16"),
    ]


def draw(rng):
    kind = rng.choice(["step", "scan", "learn", "scan", "learn", "conv", "conv", "block", "block", "update"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    starts = rng.random() < 0.6
    grad = rng.random() < 0.5
    if kind == "update":
        width = _spread(rng, 24, 2000)
        layers = rng.randint(1, max(1, min(8, int(8 * (2000 / width) ** 2))))
        return _update(None, layers, width, rng.choice(["float32", dtype]), dtype)
    if kind == "block":
        width = rng.choice([64, 192, 256, 256, 384, 512, 1000, 1024, 2048, _spread(rng, 17, 5000)])
        t = _spread(rng, 1, 2048)
        b = _spread(rng, 1, max(1, min(1024, (1 << 25) // (t * width))))
        return _block(None, b, t, width, dtype, wide_residual=rng.random() < 0.5, gate=rng.random() < 0.7,
                      scale=rng.random() < 0.7, weights=rng.random() < 0.8, grad=grad)
    if kind == "conv":
        channels = rng.choice([128, 256, 384, 384, 640, 1024, 1280, _spread(rng, 24, 2500)])
        t = rng.choice([0, _spread(rng, 1, 16384), _spread(rng, 1, 16384)])
        b = _spread(rng, 1, max(1, min(1024, (48 << 20) // (max(1, t) * channels))))
        return _conv(None, b, t, channels, rng.choice([2, 3, 4, 4, 4]), dtype, starts=starts, grad=grad and t > 0,
                     state=rng.random() < 0.5)
    groups = rng.choice([1, 1, 2, 3, 4])
    heads = groups * rng.choice([1, 2, 3, 4, 8])
    n, p = (rng.choice([16, 32, 48, 64, 64, 80, 96, 128, 128, rng.randint(9, 127)]) for _ in range(2))
    if kind == "step":
        b = _spread(rng, 1, max(1, min(1024, (1 << 26) // (heads * n * p))))
        return _step(None, b, heads, groups, n, p, dtype, starts=starts)
    grad = kind == "learn"
    t = _spread(rng, 1, 4096 if grad else 16384)
    most = min((1 << (31 if grad else 32)) // (t * heads * n * p), (1 << 26) // (t * heads * (n + p)),
               (1 << 26) // (heads * n * p))
    b = _spread(rng, 1, max(1, min(1024, most)))
    return _scan(None, b, t, heads, groups, n, p, dtype, starts=starts, state=rng.random() < 0.5, grad=grad)


def _named(name, case):
    return case if name is None else {"name": name, **case}


def _step(name, envs, heads, groups, n, p, dtype, starts=True):
    return _named(name, {"op": "step", "envs": envs, "heads": heads, "groups": groups, "state_dim": n, "head_dim": p,
                         "dtype": dtype, "starts": starts})


def _scan(name, envs, steps, heads, groups, n, p, dtype, starts=True, state=False, grad=False):
    return _named(name, {"op": "scan", "envs": envs, "steps": steps, "heads": heads, "groups": groups, "state_dim": n,
                         "head_dim": p, "dtype": dtype, "starts": starts, "state": state, "grad": grad})


def _conv(name, envs, steps, channels, taps, dtype, starts=True, state=False, grad=False):
    """``steps`` 0: the form for one frame, its window updated in place."""
    return _named(name, {"op": "conv", "envs": envs, "steps": steps, "channels": channels, "taps": taps, "dtype": dtype,
                         "starts": starts, "state": state or steps == 0, "grad": grad})


def _block(name, envs, steps, width, dtype, wide_residual=False, gate=True, scale=True, weights=True, grad=False):
    return _named(name, {"op": "block", "envs": envs, "steps": steps, "width": width, "dtype": dtype,
                         "residual_dtype": "float32" if wide_residual else dtype, "gate": gate, "scale": scale,
                         "weights": weights, "grad": grad})


def _update(name, layers, width, dtype, out_dtype):
    return _named(name, {"op": "update", "layers": layers, "width": width, "dtype": dtype, "out_dtype": out_dtype})


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _update_shapes(case):
    """The matrices of a policy of ``layers`` blocks: an encoder's first product of odd size, four
    square products, one to twice the width and one back, a head of seven actions."""
    w = case["width"]
    return [(w, 105)] + ([(w, w)] * 4 + [(2 * w, w), (w, 2 * w)]) * case["layers"] + [(7, w)]


# ---- what a user's program has in hand ----


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    return {"case": case, **_PREPARE[case["op"]](case, gen)}


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE)


def _uniform(gen, lo, hi, *shape):
    return lo + (hi - lo) * torch.rand(shape, generator=gen, device=DEVICE)


def _starts(case, gen, *lead):
    return torch.rand(lead, generator=gen, device=DEVICE) < 1.0 / 50 if case["starts"] else None


def _memory_inputs(case, gen, lead):
    """What a convolution with silu leaves (x, B, C), decay rates of 1 to 16 and steps of 0.001 to
    0.1 as such a memory is begun with, moved by what the token says; episodes that end."""
    h, g, n, p = case["heads"], case["groups"], case["state_dim"], case["head_dim"]
    dtype = TYPES[case["dtype"]]
    first = torch.exp(_uniform(gen, math.log(0.001), math.log(0.1), h))
    s = {
        "x": torch.nn.functional.silu(_randn(gen, *lead, h, p)).to(dtype),
        "dt": 0.8 * _randn(gen, *lead, h),
        "a": -_uniform(gen, 1.0, 16.0, h),
        "b": torch.nn.functional.silu(_randn(gen, *lead, g, n)).to(dtype),
        "c": torch.nn.functional.silu(_randn(gen, *lead, g, n)).to(dtype),
        "d": 1.0 + 0.2 * _randn(gen, h),
        "dt_bias": first + torch.log(-torch.expm1(-first)),
        "starts": _starts(case, gen, *lead),
    }
    if case["op"] == "step" or case["state"]:
        s["state"] = 0.3 * _randn(gen, lead[0], h, n, p)
    return s


def _prepare_step(case, gen):
    return _memory_inputs(case, gen, (case["envs"],))


def _prepare_scan(case, gen):
    s = _memory_inputs(case, gen, (case["envs"], case["steps"]))
    if case["grad"]:
        s["grad_y"] = _randn(gen, *s["x"].shape).to(s["x"].dtype)
        if case["state"]:
            s["grad_state"] = 0.3 * _randn(gen, *s["state"].shape)
        _require(s, _SCAN_INPUTS)
    return s


def _prepare_conv(case, gen):
    dtype, c, w = TYPES[case["dtype"]], case["channels"], case["taps"]
    lead = (case["envs"], case["steps"]) if case["steps"] else (case["envs"],)
    s = {
        "x": _randn(gen, *lead, c).to(dtype),
        "weight": _randn(gen, c, w) / math.sqrt(w),
        "bias": 0.1 * _randn(gen, c),
        "starts": _starts(case, gen, *lead),
    }
    if case["state"]:
        s["window"] = _randn(gen, lead[0], w - 1, c).to(dtype)
    if case["grad"]:
        s["grad_y"] = _randn(gen, *s["x"].shape).to(dtype)
        if case["state"]:
            s["grad_window"] = _randn(gen, *s["window"].shape).to(dtype)
        _require(s, _CONV_INPUTS)
    return s


def _prepare_block(case, gen):
    dtype, wide, w = TYPES[case["dtype"]], TYPES[case["residual_dtype"]], case["width"]
    lead = (case["envs"], case["steps"])
    level = torch.exp(0.5 * _randn(gen, *lead, 1))
    s = {"y": (level * _randn(gen, *lead, w)).to(dtype), "residual": (2.0 * level * _randn(gen, *lead, w)).to(wide)}
    if case["gate"]:
        s["gate"] = _randn(gen, *lead, w).to(dtype)
    if case["scale"]:
        s["scale"] = 0.5 + 0.2 * _randn(gen, w)
    if case["weights"]:
        s["post_weight"], s["pre_weight"] = (1.0 + 0.2 * _randn(gen, w) for _ in range(2))
    if case["grad"]:
        s["grad_stream"], s["grad_normed"] = _randn(gen, *lead, w).to(wide), _randn(gen, *lead, w).to(dtype)
        _require(s, _BLOCK_INPUTS)
    return s


def _prepare_update(case, gen):
    """Momenta: a part of low rank that most of the update is in, and noise."""
    dtype, out = TYPES[case["dtype"]], TYPES[case["out_dtype"]]
    updates = []
    for m, n in _update_shapes(case):
        r = max(1, min(m, n) // 8)
        low = _randn(gen, m, r) * torch.exp(_randn(gen, r)) @ _randn(gen, r, n) / math.sqrt(r)
        updates.append((1e-3 * (low + 0.5 * _randn(gen, m, n))).to(dtype))
    shapes = _update_shapes(case)
    sizes = [math.prod(x) for x in shapes]
    flat = torch.empty(sum(sizes), dtype=out, device=DEVICE)  # what the optimizer reads
    return {"updates": updates, "flat": flat, "out": [x.view(y) for x, y in zip(flat.split(sizes), shapes)]}


_PREPARE = {"step": _prepare_step, "scan": _prepare_scan, "conv": _prepare_conv, "block": _prepare_block,
            "update": _prepare_update}
_SCAN_INPUTS = ("x", "dt", "a", "b", "c", "d", "dt_bias", "state")
_CONV_INPUTS = ("x", "weight", "bias", "window")
_BLOCK_INPUTS = ("y", "residual", "gate", "scale", "post_weight", "pre_weight")


def _require(s, names):
    for x in names:
        if x in s:
            s[x].requires_grad_()


# ---- one pass ----


def run(state):
    op = state["case"]["op"]
    return _OWN[op](state) if own else _PLAIN[op](state)


def _own_step(s):
    from navi_amd import policy

    y = policy.selective_scan_step(s["x"], s["dt"], s["a"], s["b"], s["c"], s["state"], d=s["d"], dt_bias=s["dt_bias"],
                                   starts=s["starts"])
    return {"y": y, "state": s["state"]}


def _own_scan(s):
    from navi_amd import policy

    carried = s["case"]["state"]
    got = policy.selective_scan(s["x"], s["dt"], s["a"], s["b"], s["c"], d=s["d"], dt_bias=s["dt_bias"],
                                starts=s["starts"], initial_state=s.get("state"), return_state=carried)
    return _outputs(s, {"y": got[0], "state": got[1]} if carried else {"y": got}, _SCAN_INPUTS)


def _own_conv(s):
    from navi_amd import policy

    if not s["case"]["steps"]:
        y = policy.causal_conv_step(s["x"], s["weight"], s["window"], bias=s["bias"], starts=s["starts"])
        return {"y": y, "window": s["window"]}
    carried = s["case"]["state"]
    got = policy.causal_conv(s["x"], s["weight"], bias=s["bias"], starts=s["starts"], initial_window=s.get("window"),
                             return_window=carried)
    return _outputs(s, {"y": got[0], "window": got[1]} if carried else {"y": got}, _CONV_INPUTS)


def _own_block(s):
    from navi_amd import policy

    stream, normed = policy.block_norm(s["y"], s["residual"], gate=s.get("gate"), scale=s.get("scale"),
                                       post_weight=s.get("post_weight"), pre_weight=s.get("pre_weight"))
    return _outputs(s, {"stream": stream, "normed": normed}, _BLOCK_INPUTS)


def _own_update(s):
    from navi_amd import policy

    policy.orthogonalize(s["updates"], out=s["out"])
    return s["flat"]


_OWN = {"step": _own_step, "scan": _own_scan, "conv": _own_conv, "block": _own_block, "update": _own_update}


def _outputs(s, outputs, inputs):
    """The outputs, in a learner's pass with the gradients of the inputs beside them."""
    if not s["case"]["grad"]:
        return outputs
    wanted = [x for x in inputs if x in s]
    grads = torch.autograd.grad(list(outputs.values()), [s[x] for x in wanted], [s["grad_" + x] for x in outputs])
    return {**{x: y.detach() for x, y in outputs.items()}, **{"d_" + x: y for x, y in zip(wanted, grads)}}


# ---- the plain forms, in 32 bits ----


def _plain_step(s):
    h = s["case"]["heads"]
    b, c = (s[x].float().repeat_interleave(h // s["case"]["groups"], 1) for x in ("b", "c"))
    beta = torch.nn.functional.softplus(s["dt"] + s["dt_bias"])
    keep = torch.exp(beta * s["a"])
    if s["starts"] is not None:
        keep = torch.where(s["starts"][:, None], torch.zeros_like(keep), keep)
    x = s["x"].float()
    state = keep[..., None, None] * s["state"] + (beta[..., None] * b)[..., None] * x[..., None, :]
    y = (c[..., None] * state).sum(-2) + s["d"][:, None] * x
    s["state"].copy_(state)
    return {"y": y.to(s["x"].dtype), "state": s["state"]}


def _plain_scan(s):
    """In chunks: what each adds to the state, all states before a chunk by one masked product
    over the chunks, and the outputs from those and the tokens of the chunk itself."""
    c = s["case"]
    e, t, h, p = s["x"].shape
    n = -(-t // CHUNK)
    pad = n * CHUNK - t

    def chunks(x):  # [E, T, H, ...] -> [E, H, n, CHUNK, ...], zeros after the last token
        x = torch.cat([x, x.new_zeros(e, pad, *x.shape[2:])], 1) if pad else x
        return x.transpose(1, 2).reshape(e, x.shape[2], n, CHUNK, *x.shape[3:])

    values = s["x"].float()
    x = chunks(values)
    b, r = (chunks(s[y].float().repeat_interleave(h // c["groups"], 2)) for y in ("b", "c"))
    beta = torch.nn.functional.softplus(s["dt"] + s["dt_bias"])
    log = beta.double() * s["a"].double()  # sums over far tokens need differences of large numbers
    first = torch.zeros_like(log, dtype=torch.bool)
    if s["starts"] is not None:
        first = s["starts"][..., None].expand(e, t, h)
    total = chunks(torch.where(first, torch.zeros_like(log), log)).flatten(2).cumsum(-1).unflatten(2, (n, CHUNK))
    episode = chunks(first.int()).flatten(2).cumsum(-1).unflatten(2, (n, CHUNK))
    beta = chunks(beta)

    def decay(to, from_, same):
        return torch.exp((to - from_).masked_fill(~same, -math.inf)).float()

    row = torch.arange(CHUNK, device=x.device)
    within = decay(total[..., :, None], total[..., None, :],
                   (episode[..., :, None] == episode[..., None, :]) & (row[:, None] >= row))
    end, end_episode = total[..., -1], episode[..., -1]
    added = (decay(end[..., None], total, end_episode[..., None] == episode) * beta)[..., None] * b
    added = added.transpose(-1, -2) @ x  # [E, H, n, N, P]
    before = torch.nn.functional.pad(end[..., :-1], (1, 0))  # sums up to each chunk
    before_episode = torch.nn.functional.pad(end_episode[..., :-1], (1, 0))
    earlier = torch.arange(n, device=x.device)
    carry = decay(before[..., :, None], end[..., None, :],
                  (before_episode[..., :, None] == end_episode[..., None, :]) & (earlier[:, None] > earlier))
    states = (carry @ added.flatten(-2)).view_as(added)
    if c["state"]:
        states = states + decay(before, torch.zeros_like(before), before_episode == 0)[..., None, None] * s["state"][:, :, None]
    y = decay(total, before[..., None], episode == before_episode[..., None])[..., None] * (r @ states)
    y = y + (within * beta[..., None, :] * (r @ b.transpose(-1, -2))) @ x
    y = y.reshape(e, h, n * CHUNK, p)[:, :, :t].transpose(1, 2) + s["d"][:, None] * values
    out = {"y": y.to(s["x"].dtype)}
    if c["state"]:
        keep = decay(end[..., -1], before[..., -1], end_episode[..., -1] == before_episode[..., -1])
        out["state"] = keep[..., None, None] * states[:, :, -1] + added[:, :, -1]
    return _outputs(s, out, _SCAN_INPUTS)


def _plain_conv(s):
    c = s["case"]
    w, dtype = c["taps"], s["x"].dtype
    x = s["x"].float() if c["steps"] else s["x"].float()[:, None]
    e, t = x.shape[:2]
    earlier = s["window"].float() if "window" in s else x.new_zeros(e, w - 1, c["channels"])
    x = torch.cat([earlier, x], 1)
    episode = torch.zeros(e, t, dtype=torch.int64, device=x.device)
    if s["starts"] is not None:
        episode = s["starts"].view(e, t).long().cumsum(1)
    episode = torch.cat([episode.new_zeros(e, w - 1), episode], 1)
    same = episode.unfold(1, w, 1) == episode[:, w - 1:, None]
    taken = torch.where(same[:, :, None], x.unfold(1, w, 1), 0.0)
    y = torch.nn.functional.silu((taken * s["weight"]).sum(-1) + s["bias"]).to(dtype)
    window = torch.where((episode[:, t:] == episode[:, -1:])[..., None], x[:, t:], 0.0).to(dtype)
    if not c["steps"]:
        s["window"].copy_(window)
        return {"y": y[:, 0], "window": s["window"]}
    return _outputs(s, {"y": y, "window": window} if c["state"] else {"y": y}, _CONV_INPUTS)


def _plain_norm(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _plain_block(s):
    m = _plain_norm(s["y"].float())
    m = m * s["post_weight"] if "post_weight" in s else m
    m = m * torch.nn.functional.silu(s["gate"].float()) if "gate" in s else m
    m = m * s["scale"] if "scale" in s else m
    h = s["residual"].float() + m
    normed = _plain_norm(h)
    normed = normed * s["pre_weight"] if "pre_weight" in s else normed
    return _outputs(s, {"stream": h.to(s["residual"].dtype), "normed": normed.to(s["y"].dtype)}, _BLOCK_INPUTS)


def _plain_update(s):
    for g, out in zip(s["updates"], s["out"]):
        wide = g.shape[0] <= g.shape[1]
        x = g.float()
        x = x / (torch.sqrt(x.square().sum()) + EPS)
        x = x if wide else x.T
        for _ in range(STEPS):
            gram = x @ x.T
            x = FACTORS[0] * x + (FACTORS[1] * gram + FACTORS[2] * (gram @ gram)) @ x
        out.copy_(x if wide else x.T)
    return s["flat"]


_PLAIN = {"step": _plain_step, "scan": _plain_scan, "conv": _plain_conv, "block": _plain_block, "update": _plain_update}


# ---- what a pass cannot do without ----


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "update":
        shapes = [(min(x), max(x)) for x in _update_shapes(case)]
        size = sum(m * n for m, n in shapes)
        # of the symmetric products (X X', A A) one half
        return {"bytes": size * (e + BYTES[case["out_dtype"]]), "flops": STEPS * sum(3 * m * m * n + m ** 3 for m, n in shapes)}
    b, t = case["envs"], case.get("steps") or 1
    passes = 3 if case.get("grad") else 1
    mark = b * t if case.get("starts") else 0
    if case["op"] == "block":
        w, r = case["width"], BYTES[case["residual_dtype"]]
        row = w * (2 * e + 2 * r + (e if case["gate"] else 0))  # y, normed, residual, stream, gate
        if case["grad"]:  # those of the outputs in, those of the inputs out
            row += w * (2 * e + 2 * r + (e if case["gate"] else 0))
        vectors = 4 * w * (3 if case["weights"] and case["scale"] else 2 if case["weights"] else 1 if case["scale"] else 0)
        return {"bytes": b * t * row + vectors * (2 if case["grad"] else 1), "flops": 14 * b * t * w * passes}
    if case["op"] == "conv":
        n, w = b * t * case["channels"], case["taps"]
        windows = 2 * b * (w - 1) * case["channels"] * e if case["state"] else 0
        vectors = 4 * case["channels"] * (w + 1)
        total = 2 * n * e + windows + vectors + mark
        if case["grad"]:
            total += 2 * n * e + windows + vectors
        return {"bytes": total, "flops": (2 * w + 4) * n * passes}
    h, g, n, p = case["heads"], case["groups"], case["state_dim"], case["head_dim"]
    inputs = b * t * (e * (h * p + 2 * g * n) + 4 * h) + 12 * h
    out = b * t * h * p * e
    states = 4 * b * h * n * p
    flops = 5 * b * t * h * n * p * passes  # decay, update and S'C of the recurrence
    if case["op"] == "step":
        return {"bytes": inputs + out + 2 * states + mark, "flops": flops}
    total = inputs + out + mark + (2 * states if case["state"] else 0)
    if case["grad"]:
        total += out + inputs + (2 * states if case["state"] else 0)
    return {"bytes": total, "flops": flops}


# ---- the definitions in 64 bits ----


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _EXACT[case["op"]](case, {x: y.detach().double() if torch.is_tensor(y) and y.is_floating_point() else y
                                         for x, y in s.items()})


def _softplus(z):
    return torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs()))


def _exact_token(case, s, state, at):
    """One token of the recurrence: output, state after it and what its gradient needs."""
    rep = case["heads"] // case["groups"]
    z = at(s["dt"]) + s["dt_bias"]
    beta = _softplus(z)
    keep = torch.exp(beta * s["a"])
    if s["starts"] is not None:
        keep = keep * (~at(s["starts"]))[:, None]
    b, c = (at(s[x]).repeat_interleave(rep, 1) for x in ("b", "c"))
    x = at(s["x"])
    after = torch.einsum("eh,ehnp->ehnp", keep, state) + torch.einsum("ehn,ehp->ehnp", beta[..., None] * b, x)
    y = torch.einsum("ehnp,ehn->ehp", after, c) + s["d"][:, None] * x
    return y, after, (state, z, beta, keep, b, c, x)


def _exact_step(case, s):
    y, state, _ = _exact_token(case, s, s["state"], lambda x: x)
    return {"y": y, "state": state}


def _exact_scan(case, s):
    e, t, h, g, n, p = (case[x] for x in ("envs", "steps", "heads", "groups", "state_dim", "head_dim"))
    if case["grad"] and 8 * e * t * h * n * p > 70e9:
        return None  # a state for every token does not fit
    state = s["state"] if case["state"] else torch.zeros(e, h, n, p, dtype=torch.float64, device=DEVICE)
    y, tape = torch.empty_like(s["x"]), []
    for i in range(t):
        y[:, i], state, rest = _exact_token(case, s, state, lambda x: x[:, i])
        if case["grad"]:
            tape.append(rest)
    got = {"y": y, **({"state": state} if case["state"] else {})}
    if not case["grad"]:
        return got
    d = {x: torch.zeros_like(s[x]) for x in _SCAN_INPUTS if x in s}
    ds = s["grad_state"].clone() if case["state"] else torch.zeros_like(state)
    after = state
    for i in reversed(range(t)):
        before, z, beta, keep, b, c, x = tape.pop()
        dy = s["grad_y"][:, i]
        ds = ds + torch.einsum("ehn,ehp->ehnp", c, dy)
        dx = torch.einsum("ehnp,ehn->ehp", ds, b)
        dlog = keep * (before * ds).sum((-1, -2))
        dbeta = (dx * x).sum(-1) + dlog * s["a"]
        d["c"][:, i] = torch.einsum("ehnp,ehp->ehn", after, dy).view(e, g, h // g, n).sum(2)
        d["b"][:, i] = (beta[..., None] * torch.einsum("ehnp,ehp->ehn", ds, x)).view(e, g, h // g, n).sum(2)
        d["x"][:, i] = beta[..., None] * dx + s["d"][:, None] * dy
        d["dt"][:, i] = dbeta * torch.sigmoid(z)
        d["a"] += (dlog * beta).sum(0)
        d["d"] += (dy * x).sum((0, 2))
        ds, after = keep[..., None, None] * ds, before
    d["dt_bias"] = d["dt"].sum((0, 1))
    if case["state"]:
        d["state"] = ds
    return {**got, **{"d_" + x: y for x, y in d.items()}}


def _exact_conv(case, s):
    e, w, c = case["envs"], case["taps"], case["channels"]
    t = case["steps"] or 1
    x = s["x"].view(e, t, c)
    starts = s["starts"].view(e, t) if s["starts"] is not None else torch.zeros(e, t, dtype=torch.bool, device=DEVICE)
    # steps since the episode began (many, before the first start)
    place = torch.arange(t, device=DEVICE)
    since = place - torch.where(starts, place, -w).cummax(1).values
    source = torch.cat([s["window"] if "window" in s else x.new_zeros(e, w - 1, c), x], 1)
    z = s["bias"].expand(e, t, c).clone()
    for back in range(w):
        z += s["weight"][:, w - 1 - back] * (source[:, w - 1 - back:w - 1 - back + t] * (since >= back)[..., None])
    sigma = torch.sigmoid(z)
    kept = torch.stack([since[:, -1] >= back for back in reversed(range(w - 1))], 1)[..., None] if w > 1 else None
    window = source[:, t:] * kept if w > 1 else source[:, t:]
    if not case["steps"]:
        return {"y": (z * sigma)[:, 0], "window": window}
    got = {"y": z * sigma, **({"window": window} if case["state"] else {})}
    if not case["grad"]:
        return got
    dz = s["grad_y"] * sigma * (1 + z * (1 - sigma))
    dsource, dweight = torch.zeros_like(source), torch.zeros_like(s["weight"])
    if case["state"]:
        dsource[:, t:] += s["grad_window"] * kept
    for back in range(w):
        reached = dz * (since >= back)[..., None]
        at = slice(w - 1 - back, w - 1 - back + t)
        dsource[:, at] += s["weight"][:, w - 1 - back] * reached
        dweight[:, w - 1 - back] = (reached * source[:, at]).sum((0, 1))
    got.update({"d_x": dsource[:, w - 1:], "d_weight": dweight, "d_bias": dz.sum((0, 1))})
    return {**got, "d_window": dsource[:, :w - 1]} if case["state"] else got


def _exact_block(case, s):
    one = torch.ones((), dtype=torch.float64, device=DEVICE)
    post, pre, scale = (s.get(x, one) for x in ("post_weight", "pre_weight", "scale"))
    w = case["width"]
    r1 = 1 / torch.sqrt((s["y"] ** 2).sum(-1, keepdim=True) / w + EPS)
    n1 = s["y"] * r1
    sigma = torch.sigmoid(s["gate"]) if case["gate"] else one
    gate = s["gate"] * sigma if case["gate"] else one
    m = n1 * post * gate
    h = s["residual"] + scale * m
    r2 = 1 / torch.sqrt((h ** 2).sum(-1, keepdim=True) / w + EPS)
    got = {"stream": h, "normed": h * r2 * pre}
    if not case["grad"]:
        return got
    dn = s["grad_normed"] * pre
    dh = s["grad_stream"] + r2 * dn - h * r2 ** 3 * (dn * h).sum(-1, keepdim=True) / w
    dz = scale * dh * gate
    dn1 = dz * post
    got["d_y"] = r1 * dn1 - s["y"] * r1 ** 3 * (dn1 * s["y"]).sum(-1, keepdim=True) / w
    got["d_residual"] = dh
    if case["gate"]:
        got["d_gate"] = scale * dh * n1 * post * sigma * (1 + s["gate"] * (1 - sigma))
    if case["scale"]:
        got["d_scale"] = (dh * m).sum((0, 1))
    if case["weights"]:
        got["d_post_weight"] = (dz * n1).sum((0, 1))
        got["d_pre_weight"] = (s["grad_normed"] * h * r2).sum((0, 1))
    return got


def _exact_update(case, s):
    a, b, c = FACTORS
    got = []
    for g in s["updates"]:
        x = g.double()
        wide = x.shape[0] <= x.shape[1]
        x = x / (torch.linalg.vector_norm(x) + EPS)
        x = x.T if wide else x  # the tall one, and its small Gram matrix on the other side
        for _ in range(STEPS):
            gram = x.T @ x
            x = a * x + x @ (gram @ (b * torch.eye(len(gram), dtype=x.dtype, device=x.device) + c * gram))
        got.append((x.T if wide else x).reshape(-1))
    return torch.cat(got)


_EXACT = {"step": _exact_step, "scan": _exact_scan, "conv": _exact_conv, "block": _exact_block, "update": _exact_update}

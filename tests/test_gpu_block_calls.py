"""How a block's operators (convolution, selective scan, block norms, orthogonalised updates) are called:
arguments that are refused, writes that autograd is told of, derivatives that they do not have, streams,
threads, graphs. Equal calls give equal bits: results are compared exactly."""

from __future__ import annotations

import threading

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def policy(gpu):
    from navi_amd import policy

    return policy


ENVS, HEADS, GROUPS, DIM, WIDE, TAPS = 3, 4, 2, 16, 24, 4
CHANNELS = HEADS * WIDE


def inputs(steps=70, dtype=torch.float32, seed=0):
    """Inputs of a rollout for each operator, by its arguments' names."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    lead = (ENVS, steps)
    starts = torch.rand(*lead, generator=gen, device="cuda") < 0.1
    return {
        "selective_scan": dict(
            x=rand(*lead, HEADS, WIDE).to(dtype), dt=rand(*lead, HEADS) - 2, a=-rand(HEADS).abs(),
            b=rand(*lead, GROUPS, DIM).to(dtype), c=rand(*lead, GROUPS, DIM).to(dtype), d=rand(HEADS), dt_bias=rand(HEADS),
            starts=starts, initial_state=rand(ENVS, HEADS, DIM, WIDE)),
        "causal_conv": dict(x=rand(*lead, CHANNELS).to(dtype), weight=rand(CHANNELS, TAPS), bias=rand(CHANNELS), starts=starts,
                            initial_window=rand(ENVS, TAPS - 1, CHANNELS).to(dtype)),
        "block_norm": dict(y=rand(*lead, CHANNELS).to(dtype), residual=rand(*lead, CHANNELS), gate=rand(*lead, CHANNELS).to(dtype),
                           scale=rand(CHANNELS), post_weight=rand(CHANNELS), pre_weight=rand(CHANNELS)),
    }


def frame(name, given):
    """The step's arguments for a rollout's first frame: (positional, keywords, what is carried)."""
    at = {n: t[:, 0].contiguous() if n in ("x", "dt", "b", "c", "starts") else t for n, t in given.items()}
    if name == "selective_scan":
        state = at["initial_state"].clone()
        return [at[n] for n in ("x", "dt", "a", "b", "c")] + [state], {n: at[n] for n in ("d", "dt_bias", "starts")}, state
    window = at["initial_window"].clone()
    return [at["x"], at["weight"], window], {n: at[n] for n in ("bias", "starts")}, window


STEPS = ["selective_scan", "causal_conv"]


def step_of(policy, name):
    return getattr(policy, name + "_step")


def matrices(seed=0, dtype=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(m, n, generator=gen, device="cuda").to(dtype) for m, n in ((40, 96), (96, 40), (64, 64), (130, 7))]


def together(policy, given, updates=None):
    """All the operators' results, one list."""
    got = [*policy.selective_scan(**given["selective_scan"], return_state=True),
           *policy.causal_conv(**given["causal_conv"], return_window=True), *policy.block_norm(**given["block_norm"])]
    if updates is not None:
        out = [torch.empty_like(u) for u in updates]
        policy.orthogonalize(updates, out=out)
        got += out
    return got


def backward(policy, given, ones=torch.ones_like):
    """Gradients of every operator in all its inputs, through leaves of this call."""
    grads = []
    for name, args in given.items():
        leaves = {n: t.detach().requires_grad_(t.is_floating_point()) for n, t in args.items()}
        outs = getattr(policy, name)(**leaves, **({} if name == "block_norm" else
                                                  {"return_state" if name == "selective_scan" else "return_window": True}))
        wanted = [t for t in leaves.values() if t.requires_grad]
        grads += torch.autograd.grad(outs, wanted, [ones(o) for o in outs])
    return grads


# ---- what is refused ----


def ragged(t):
    """The same numbers, two apart."""
    return torch.stack([t, t], -1).flatten(-2)[..., ::2]


WRONG = [
    ("selective_scan", "x", lambda t: t.double(), "x must be"),
    ("selective_scan", "x", lambda t: t[0], "dimensions"),
    ("selective_scan", "x", ragged, "x must be contiguous in its last dimension"),
    ("selective_scan", "b", lambda t: t.half(), "b must be float32"),
    ("selective_scan", "b", lambda t: t[:, :-1], "b and c must both be"),
    ("selective_scan", "c", lambda t: t[..., :-1], "b and c must both be"),
    ("selective_scan", "c", lambda t: t.cpu(), "c must be a CUDA tensor"),
    ("selective_scan", "dt", lambda t: t.bfloat16(), "dt must be float32"),
    ("selective_scan", "dt", lambda t: t[..., :-1], "dt must be"),
    ("selective_scan", "a", lambda t: None, "a must be a CUDA tensor"),
    ("selective_scan", "a", lambda t: t[:-1], "a must be"),
    ("selective_scan", "d", lambda t: t.half(), "d must be float32"),
    ("selective_scan", "dt_bias", lambda t: ragged(t), "dt_bias must be"),
    ("selective_scan", "starts", lambda t: t.float(), "starts must be"),
    ("selective_scan", "starts", lambda t: t[:, :-1], "starts must be"),
    ("selective_scan", "initial_state", lambda t: t[:-1], "initial_state must be"),
    ("selective_scan", "initial_state", lambda t: t.transpose(2, 3).contiguous().transpose(2, 3), "initial_state must be contiguous"),
    ("causal_conv", "x", lambda t: t.double(), "x must be"),
    ("causal_conv", "x", ragged, "x must be contiguous in its last dimension"),
    ("causal_conv", "weight", lambda t: t.half(), "weight must be float32"),
    ("causal_conv", "weight", lambda t: t[:, :1].contiguous(), "with 2 to 4 taps"),
    ("causal_conv", "weight", lambda t: torch.cat([t, t], 1), "with 2 to 4 taps"),
    ("causal_conv", "weight", lambda t: t.T.contiguous().T, "weight must be"),
    ("causal_conv", "bias", lambda t: t[:-1], "bias must be"),
    ("causal_conv", "starts", lambda t: t.int(), "starts must be"),
    ("causal_conv", "initial_window", lambda t: t[:, 1:], "initial_window must be"),
    ("causal_conv", "initial_window", lambda t: t.half(), "initial_window must be"),
    ("block_norm", "y", lambda t: t.double(), "y must be"),
    ("block_norm", "y", lambda t: t[0], "dimensions"),
    ("block_norm", "y", ragged, "contiguous in its last dimension"),
    ("block_norm", "residual", lambda t: t.half(), "residual must be"),
    ("block_norm", "residual", lambda t: t[:, 1:], "residual must be"),
    ("block_norm", "gate", lambda t: t.half(), "gate must be"),
    ("block_norm", "gate", lambda t: t[..., 1:], "gate must be"),
    ("block_norm", "scale", lambda t: t[1:], "scale must be"),
    ("block_norm", "pre_weight", lambda t: t.cpu(), "pre_weight must be"),
]


@pytest.mark.parametrize("name, argument, change, words", WRONG, ids=[f"{i}-{w[0]}-{w[1]}" for i, w in enumerate(WRONG)])
def test_refusals(policy, name, argument, change, words):
    given = inputs()[name]
    with pytest.raises(RuntimeError, match=words):
        getattr(policy, name)(**{**given, argument: change(given[argument])})


def test_refusals_of_groups_activations_and_eps(policy):
    given = inputs()
    scan = given["selective_scan"]
    three = torch.cat([scan["b"], scan["b"][:, :, :1]], 2)
    with pytest.raises(RuntimeError, match="multiple of the groups"):
        policy.selective_scan(**{**scan, "b": three, "c": three})
    for activation in ("gelu", 1, ["silu"], torch.ones(2)):
        with pytest.raises(RuntimeError, match="activation must be"):
            policy.causal_conv(**given["causal_conv"], activation=activation)
    for eps in (-1e-6, float("nan"), float("inf"), 1e39):
        with pytest.raises(RuntimeError, match="eps must be"):
            policy.block_norm(**given["block_norm"], eps=eps)


@pytest.mark.parametrize("name", STEPS)
def test_refusals_of_steps(policy, name):
    args, more, carried = frame(name, inputs()[name])
    step, kept = step_of(policy, name), carried.clone()
    out = torch.empty_like(args[0])
    whole = torch.empty(2, *out.shape, device="cuda")
    for wrong, words in ((out.half(), "out must be"), (out[1:], "out must be"), (ragged(out), "out must be"), (out.cpu(), "out must be"),
                         (carried.flatten()[:out.numel()].view_as(out), "shares memory")):
        with pytest.raises(RuntimeError, match=words):
            step(*args, **more, out=wrong)
    shared = whole.flatten()[1:1 + out.numel()].view_as(out)
    moved = whole.flatten()[:out.numel()].view_as(out).copy_(args[0])
    with pytest.raises(RuntimeError, match="shares memory"):
        step(moved, *args[1:], **more, out=shared)
    with pytest.raises(RuntimeError, match="must be"):
        step(*args[:-1], carried[1:], **more)
    with pytest.raises(RuntimeError, match="contiguous"):
        step(*args[:-1], carried.transpose(-1, -2).contiguous().transpose(-1, -2), **more)
    assert torch.equal(carried, kept)


def test_refusals_of_matrices(policy):
    g = torch.randn(8, 12, device="cuda")
    for bad, words in (([], "at least one"), ([None], "at least one"), ([g[0]], "must be matrices"), ([g.double()], "must be float32"),
                       ([g, g.cpu()], "CUDA"), ([g.to_sparse()], "dense"), ([g, g], "share memory"), ([g, g[2:]], "share memory"),
                       ([ragged(g)], "contiguous along"), ([torch.zeros(1, 12, device="cuda").expand(8, 12)], "overlap")):
        with pytest.raises(RuntimeError, match=words):
            policy.orthogonalize(bad)
    for out, words in (([], "as long as"), ([g[1:]], "like updates"), ([g.double()], "like updates"), ([g.cpu()], "like updates")):
        with pytest.raises(RuntimeError, match=words):
            policy.orthogonalize([g], out=out)
    other = torch.randn(8, 12, device="cuda")
    with pytest.raises(RuntimeError, match="share memory"):
        policy.orthogonalize([g, other], out=[other, torch.empty_like(g)])
    for more in (dict(steps=0), dict(steps=101), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=1e39), dict(factors=(1.0, float("inf"), 0.0)),
                 dict(factors=(1.0, 0.0, -1e39))):
        with pytest.raises(RuntimeError):
            policy.orthogonalize([g], **more)


# ---- autograd ----


@pytest.mark.parametrize("name", STEPS)
def test_a_step_into_what_autograd_has_saved(policy, name):
    args, more, carried = frame(name, inputs()[name])
    step, out = step_of(policy, name), torch.empty_like(args[0])
    for written in (out, carried):
        y = (written * torch.randn_like(written).requires_grad_()).sum()
        version = written._version
        step(*args, **more, out=out)
        assert written._version > version
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_matrices_that_autograd_has_saved(policy):
    g = matrices()[0]
    y = (g * torch.ones_like(g).requires_grad_()).sum()
    policy.orthogonalize([g])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("name", STEPS)
def test_steps_have_no_gradients(policy, name):
    args, more, carried = frame(name, inputs()[name])
    step, kept = step_of(policy, name), carried.clone()
    for i in range(len(args)):
        with pytest.raises(RuntimeError, match="no gradients"):
            step(*args[:i], args[i].clone().requires_grad_(), *args[i + 1:], **more)
    with pytest.raises(RuntimeError, match="no gradients"):
        step(*args, **more, out=torch.empty_like(args[0]).requires_grad_())
    assert torch.equal(carried, kept)
    want = step(*args[:-1], kept.clone(), **more)
    with torch.no_grad():
        got = step(*[t.clone().requires_grad_() for t in args], **more)
    assert not got.requires_grad and torch.equal(got, want)


@pytest.mark.parametrize("name", ["selective_scan", "causal_conv", "block_norm"])
def test_forward_mode_is_refused(policy, name):
    given = inputs()[name]
    with forward_ad.dual_level():
        for n, t in given.items():
            if t.is_floating_point():
                with pytest.raises(RuntimeError, match="forward-mode"):
                    getattr(policy, name)(**{**given, n: forward_ad.make_dual(t, torch.ones_like(t))})
        getattr(policy, name)(**given)  # (none of its own inputs is one)
        if name in STEPS:
            args, more, _ = frame(name, given)
            for i, t in enumerate(args):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    step_of(policy, name)(*args[:i], forward_ad.make_dual(t, torch.ones_like(t)), *args[i + 1:], **more)
    if name == "block_norm":
        g = matrices()[0]
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            policy.orthogonalize([forward_ad.make_dual(g, torch.ones_like(g))])


@pytest.mark.parametrize("name", ["selective_scan", "causal_conv", "block_norm"])
def test_gradients_have_no_gradients(policy, name):
    """A second derivative is an error where it is asked for; a first one with its graph kept is the same numbers."""
    given = {n: t.requires_grad_(t.is_floating_point()) for n, t in inputs()[name].items()}
    leaves = [t for t in given.values() if t.requires_grad]

    def loss():
        out = getattr(policy, name)(**given)
        return (out[0] if name == "block_norm" else out).square().sum()

    first = torch.autograd.grad(loss(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(loss(), leaves)))
    with pytest.raises(RuntimeError, match="no gradients of their own"):
        sum(g.sum() for g in first).backward()


def test_a_second_pass_through_a_graph_is_an_error(policy):
    x = inputs()["causal_conv"]["x"].requires_grad_()
    y = policy.causal_conv(x, inputs()["causal_conv"]["weight"])
    y.sum().backward(retain_graph=True)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    assert x.grad is not None


def test_an_input_that_changes_before_the_backward_pass(policy):
    for name, args in inputs().items():
        leaves = {n: t.requires_grad_() if t.is_floating_point() else t for n, t in args.items()}
        out = getattr(policy, name)(**leaves)
        with torch.no_grad():
            next(iter(leaves.values())).mul_(2.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            (out[0] if name == "block_norm" else out).sum().backward()


def test_inference_tensors(policy):
    want = together(policy, inputs(), matrices())
    with torch.inference_mode():
        given = inputs()
        got = together(policy, given, matrices())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for name in STEPS:
            args, more, _ = frame(name, given[name])
            step_of(policy, name)(*args, **more, out=args[0])


class Named(torch.Tensor):
    """A class of a user's own."""


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_calls_in_one_step_and_by_parts_are_the_same(policy, dtype, monkeypatch):
    """The extension's calls against those that it leaves to Python."""
    given = inputs(dtype=dtype)

    def run(change=lambda t: t):
        made = []
        for name in STEPS:
            for out in (False, True):
                for rest in (True, False):
                    args, more, carried = frame(name, given[name])
                    more = more if rest else {}
                    args = [change(t) for t in args]
                    got = step_of(policy, name)(*args, **more, out=args[0] if out else None)
                    assert (got is args[0]) == out
                    made += [got, args[-1]]
        made += policy.block_norm(**{n: change(t) for n, t in given["block_norm"].items()}, eps=1e-5)
        made += policy.block_norm(change(given["block_norm"]["y"]), given["block_norm"]["residual"])
        for name in STEPS:
            args = {n: change(t) for n, t in given[name].items()}
            short = {n: t[:, :3] if n in ("x", "dt", "b", "c", "starts") else t for n, t in args.items()}
            more = {"return_state" if name == "selective_scan" else "return_window": True}
            for a in (args, short):
                made += getattr(policy, name)(**a, **more)
            leaves = {n: t.detach().requires_grad_(t.is_floating_point()) for n, t in given[name].items()}
            out, after = getattr(policy, name)(**{n: change(t) for n, t in leaves.items()}, **more)
            wanted = [t for t in leaves.values() if t.requires_grad]
            made += torch.autograd.grad([out, after], wanted, [torch.ones_like(out), torch.ones_like(after)])
        return made

    want, leaves = run(), run(lambda t: t.as_subclass(Named))

    class Leaves:
        selective_step = conv_step = selective_scan = causal_conv = block_norm = staticmethod(lambda *_: None)
        scan, conv, block = (staticmethod(getattr(policy._native.calls, n)) for n in ("scan", "conv", "block"))

    monkeypatch.setattr(policy._native, "calls", Leaves)
    for a, b, c in zip(want, run(), leaves):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and a.is_contiguous()
        assert torch.equal(a, b) and torch.equal(a, c)


def test_frames_are_read_where_they_lie(policy):
    """Strided views and odd addresses in calls of one frame."""
    for dtype in (torch.float32, torch.bfloat16):
        given = inputs(dtype=dtype)
        for name in STEPS:
            args, more, carried = frame(name, given[name])
            want = step_of(policy, name)(*args, **more)
            again, _, _ = frame(name, given[name])
            moved = [t if i in (2, len(args) - 1) or name == "causal_conv" and i == 1 else
                     torch.cat([t.flatten(1), t.flatten(1)[:, :1], t.flatten(1)], 1)[:, 1 + t.flatten(1).shape[1]:].unflatten(1, t.shape[1:])
                     for i, t in enumerate(again)]
            got = step_of(policy, name)(*moved, **more)
            assert torch.equal(got, want) and torch.equal(moved[-1], carried)


def negated(t):
    """The same numbers as a lazily negated view (the imaginary part of a conjugate)."""
    z = torch.view_as_complex(torch.stack([torch.zeros_like(t), -t], -1)).conj().imag
    assert z.is_neg() and torch.equal(z, t)
    return z


def test_lazily_negated_views(policy):
    """Their memory holds the negative: they are resolved, or refused where something is written."""
    given = inputs()
    for name, args in given.items():
        for n in ("x", "y", "gate", "dt", "b"):
            if n in args:
                got, want = (getattr(policy, name)(**{**args, n: t}) for t in (negated(args[n]).contiguous() if n in "xyb" else args[n], args[n]))
                assert all(torch.equal(p, q) for p, q in zip(*([r] if torch.is_tensor(r) else r for r in (got, want))))
    args = given["selective_scan"]
    assert torch.equal(policy.selective_scan(**{**args, "a": negated(args["a"]).clone(), "dt": negated(args["dt"])}), policy.selective_scan(**args))
    block = given["block_norm"]
    x = block["y"].clone().requires_grad_()
    s, n = policy.block_norm(x, block["residual"])
    got, want = (torch.autograd.grad([s, n], x, [g, g], retain_graph=True)[0] for g in (negated(torch.ones_like(s)), torch.ones_like(s)))
    assert torch.equal(got, want)
    for name in STEPS:
        args, more, carried = frame(name, given[name])
        if name == "selective_scan":
            with pytest.raises(RuntimeError, match="negated"):
                step_of(policy, name)(args[0], negated(args[1]), *args[2:], **more)
    g = matrices()[0]
    z = torch.view_as_complex(torch.stack([g, g], -1)).conj().imag
    with pytest.raises(RuntimeError, match="negated|contiguous"):
        policy.orthogonalize([z])


def test_matrices_that_require_grad(policy):
    g = matrices()[0]
    want = torch.empty_like(g)
    policy.orthogonalize([g], out=[want])
    leaf, kept = g.clone().requires_grad_(), g.clone()
    for updates, out in (([leaf], None), ([g], [leaf]), ([leaf * 1.0], None)):
        with pytest.raises(RuntimeError, match="no gradients"):
            policy.orthogonalize(updates, out=out)
    assert torch.equal(leaf, kept)
    with torch.no_grad():
        policy.orthogonalize([leaf])
    assert torch.equal(leaf, want)


# ---- streams, threads, graphs ----


def test_two_streams_and_threads(policy):
    given = [(inputs(seed=s, dtype=torch.bfloat16), matrices(s)) for s in (1, 2)]
    want = [together(policy, *g) + backward(policy, g[0]) for g in given]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got = together(policy, *given[i]) + backward(policy, given[i][0])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
        except Exception as error:  # noqa: BLE001 (told to the test's own thread)
            wrong.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    streams, got = [torch.cuda.Stream() for _ in given], [[], []]
    for _ in range(3):
        for i, g in enumerate(given):
            with torch.cuda.stream(streams[i]):
                got[i].append(together(policy, *g))
    for i, stream in enumerate(streams):
        stream.synchronize()
        assert all(torch.equal(a, b) for o in got[i] for a, b in zip(o, want[i]))


def refreshed(given, updates, seed):
    other = inputs(seed=seed, steps=given["causal_conv"]["x"].shape[1], dtype=given["causal_conv"]["x"].dtype)
    for name, args in given.items():
        for n, t in args.items():
            t.copy_(other[name][n])
    for t, o in zip(updates, matrices(seed)):
        t.copy_(o)


@pytest.mark.parametrize("steps", [70, 1500])  # (one part, several parts of a walk)
def test_two_graphs_replayed_in_turn(policy, steps):
    """Each replay, with eager calls and synchronizations between them, gives the eager call's bits."""
    sets = [(inputs(steps=steps, seed=s, dtype=torch.bfloat16), matrices(s)) for s in (1, 2)]
    for s in sets:
        together(policy, *s)
    torch.cuda.synchronize()
    graphs, got = [torch.cuda.CUDAGraph() for _ in sets], []
    for graph, s in zip(graphs, sets):
        with torch.cuda.graph(graph):
            got.append(together(policy, *s))
    for n in range(3):
        for i in (0, 1):
            refreshed(*sets[i], seed=10 + 2 * n + i)
        want = [together(policy, *s) for s in sets]
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), n


def test_a_captured_backward_pass(policy):
    """Forward and backward in one graph, of leaves that no eager graph holds."""
    given = inputs(seed=3, steps=130, dtype=torch.bfloat16)
    updates = []
    backward(policy, given)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = backward(policy, given)
    for n in range(3):
        refreshed(given, updates, seed=20 + n)
        want = backward(policy, given)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), n


@pytest.mark.parametrize("name", STEPS)
def test_captured_frames_replay(policy, name):
    args, more, carried = frame(name, inputs(dtype=torch.bfloat16)[name])
    begin, out = carried.clone(), torch.empty_like(args[0])
    xs = [torch.randn_like(args[0]) for _ in range(4)]
    want = [step_of(policy, name)(x, *args[1:], **more) for x in xs]
    last = carried.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step_of(policy, name)(*args, **more, out=out)
    carried.copy_(begin)
    for x, w in zip(xs, want):
        args[0].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    assert torch.equal(carried, last)


# ---- the same input twice ----


def test_inputs_that_are_one_tensor(policy):
    """b and c, x and out, y, residual and gate in one place: gradients add up."""
    given = inputs()["selective_scan"]
    b = given["b"].clone().requires_grad_()
    y = policy.selective_scan(**{**given, "b": b, "c": b})
    one = torch.autograd.grad(y, b, torch.ones_like(y))[0]
    p, q = (given["b"].clone().requires_grad_() for _ in range(2))
    z = policy.selective_scan(**{**given, "b": p, "c": q})
    two = torch.autograd.grad(z, [p, q], torch.ones_like(z))
    assert torch.equal(y, z) and torch.equal(one, two[0] + two[1])
    h = torch.randn(2, 5, 32, device="cuda").requires_grad_()
    s, n = policy.block_norm(h, h, gate=h)
    one = torch.autograd.grad([s, n], h, [torch.ones_like(s)] * 2)[0]
    each = [h.detach().clone().requires_grad_() for _ in range(3)]
    s2, n2 = policy.block_norm(each[0], each[1], gate=each[2])
    three = torch.autograd.grad([s2, n2], each, [torch.ones_like(s)] * 2)
    assert torch.equal(s, s2) and torch.equal(n, n2)
    # (two float32 sums in either order: half a step of each)
    assert torch.allclose(one, sum(three), rtol=2.0 ** -22, atol=2.0 ** -22 * float(torch.stack(three).abs().max()))


def test_broadcast_inputs(policy):
    """Frames and groups that are one in memory (expanded axes): the same results, gradients of what is expanded."""
    given = inputs(steps=90)["selective_scan"]
    b1 = given["b"][:, :, :1].clone().requires_grad_()
    args = {**given, "b": b1.expand(-1, -1, GROUPS, -1)}
    y = policy.selective_scan(**args)
    copied = b1.detach().expand(-1, -1, GROUPS, -1).contiguous().requires_grad_()
    z = policy.selective_scan(**{**given, "b": copied})
    assert torch.equal(y, z)
    got, want = torch.autograd.grad(y, b1, torch.ones_like(y))[0], torch.autograd.grad(z, copied, torch.ones_like(z))[0]
    assert torch.equal(got, want.sum(2, keepdim=True))
    same = given["x"][:, :1].expand(-1, 90, -1, -1)
    assert torch.equal(policy.selective_scan(**{**given, "x": same}), policy.selective_scan(**{**given, "x": same.contiguous()}))
    conv = inputs(steps=90)["causal_conv"]
    same = conv["x"][:, :1].expand(-1, 90, -1)
    assert torch.equal(policy.causal_conv(**{**conv, "x": same}), policy.causal_conv(**{**conv, "x": same.contiguous()}))
    block = inputs()["block_norm"]
    row = block["y"][:1, :1].expand_as(block["y"])
    assert all(torch.equal(p, q) for p, q in zip(policy.block_norm(**{**block, "y": row}), policy.block_norm(**{**block, "y": row.contiguous()})))
    y = policy.selective_scan(**{**given, "x": given["x"].clone().requires_grad_()})
    y.sum().backward()  # (a gradient that is one number everywhere)

"""What the causal mixer's operators refuse of tensors on the GPU (nothing is launched), what autograd may ask of them, streams and captured graphs."""
import pytest
import torch

import causal_reference as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _conv_args(gpu):
    return {"x": torch.randn(2, 9, 16, device=gpu), "weight": torch.randn(16, 4, device=gpu), "bias": torch.randn(16, device=gpu), "state": torch.randn(2, 3, 16, device=gpu)}


def _scan_args(gpu, B=2, L=9, C=16, N=4, G=2):
    r = lambda *s: torch.randn(*s, device=gpu)      # noqa: E731
    return {"x": r(B, L, C), "dt": r(B, L, C), "A": -torch.rand(C, N, device=gpu), "B": r(B, L, G, N), "C": r(B, L, G, N), "D": r(C), "z": r(B, L, C), "dt_bias": r(C), "state": r(B, C, N)}


def test_refused_tensors(gpu):
    import m2_amd
    a = _conv_args(gpu)
    good = m2_amd.causal_conv(**a)
    for name, bad, error in (("x", a["x"].half(), TypeError), ("x", a["x"][0], ValueError), ("x", a["x"][:, :0], ValueError), ("x", a["x"].cpu(), RuntimeError), ("x", a["x"].to_sparse(), TypeError),
                             ("weight", a["weight"].to(BF16), TypeError), ("weight", a["weight"][:8], ValueError), ("weight", torch.randn(16, 9, device=gpu), ValueError),
                             ("weight", torch.randn(16, 0, device=gpu), ValueError), ("weight", a["weight"].cpu(), RuntimeError), ("bias", a["bias"][:8], ValueError), ("bias", a["bias"].double(), TypeError),
                             ("state", a["state"][:, :2], ValueError), ("state", a["state"].to(BF16), TypeError), ("lengths", torch.ones(2, device=gpu, dtype=torch.int32), TypeError),
                             ("lengths", torch.ones(3, device=gpu, dtype=torch.int64), ValueError), ("lengths", torch.ones(2, dtype=torch.int64), RuntimeError)):
        with pytest.raises(error, match=name):
            m2_amd.causal_conv(**dict(a, **{name: bad}))
    s = _scan_args(gpu)
    again = m2_amd.selective_scan(**s)
    for name, bad, error in (("x", s["x"].half(), TypeError), ("x", s["x"][:, :0], ValueError), ("dt", s["dt"].to(BF16), TypeError), ("dt", s["dt"][:, :5], ValueError), ("A", s["A"][:5], ValueError),
                             ("A", s["A"].to(BF16), TypeError), ("A", -torch.rand(16, 257, device=gpu), ValueError), ("A", -torch.rand(16, 0, device=gpu), ValueError), ("B", s["B"][..., :3], ValueError),
                             ("B", torch.randn(2, 9, 3, 4, device=gpu), ValueError), ("B", torch.randn(2, 9, device=gpu), ValueError), ("C", s["C"][:, :, 0], ValueError), ("C", s["C"].to(BF16), TypeError),
                             ("D", s["D"][:3], ValueError), ("z", s["z"][:1], ValueError), ("dt_bias", s["dt_bias"].cpu(), RuntimeError), ("state", s["state"].to(BF16), TypeError),
                             ("state", s["state"][:1], ValueError)):
        with pytest.raises(error, match=name):
            m2_amd.selective_scan(**dict(s, **{name: bad}))
    x = torch.randn(3, 5, 16, device=gpu)
    for args, error in (((x.half(), 4), TypeError), ((x, 3), ValueError), ((x, 0), ValueError), ((x, -4), ValueError), ((x[0, 0], 4), ValueError), ((x[:, :0], 4), ValueError), ((x, 4, x[0, 0, :8]), ValueError),
                        ((x, 4, x[0, 0].to(BF16)), TypeError), ((x, 4, None, x[0, 0].cpu()), RuntimeError), ((x, 4, None, None, -1.0), ValueError), ((x, 4.0), TypeError)):
        with pytest.raises(error):
            m2_amd.group_norm(*args)
    torch.cuda.synchronize()
    assert torch.equal(m2_amd.causal_conv(**a), good) and torch.equal(m2_amd.selective_scan(**s), again)


def test_refused_steps(gpu):
    import m2_amd
    a = _conv_args(gpu)
    x, state, w = a["x"][:, 0], a["state"], a["weight"]
    big = torch.randn(2, 6, 16, device=gpu)
    for kwargs in ({"state": big[:, ::2]}, {"out_state": big[:, ::2]}, {"out_state": state[:1]}, {"state": big.view(-1)[:96].view(2, 3, 16), "out_state": big.view(-1)[16:112].view(2, 3, 16)},
                   {"x": state[:, 0]}, {"x": big[:, 1], "out_state": big.view(-1)[:96].view(2, 3, 16)}):
        args = dict({"x": x, "state": state, "weight": w}, **kwargs)
        kept = args["state"].clone()
        with pytest.raises(ValueError):
            m2_amd.causal_conv_step(**args)
        assert torch.equal(args["state"], kept)
    with pytest.raises(TypeError):
        m2_amd.causal_conv_step(x, None, w)
    with pytest.raises(TypeError):
        m2_amd.causal_conv_step(x, state, w, out_state=state.to(BF16))
    s = {k: v[:, 0] if k in ("x", "dt", "B", "C", "z") else v for k, v in _scan_args(gpu).items()}
    wide = torch.zeros(2, 16, 8, device=gpu)
    for kwargs in ({"state": wide[..., ::2]}, {"state": wide[..., :4]}, {"out_state": wide[..., :4]}, {"out_state": s["state"].view(-1)[:64].view(1, 16, 4)}):
        with pytest.raises(ValueError):
            m2_amd.selective_scan_step(**dict(s, **kwargs))
    with pytest.raises(TypeError):
        m2_amd.selective_scan_step(**dict(s, state=s["state"].to(BF16)))
    with pytest.raises(TypeError):
        m2_amd.selective_scan_step(**dict(s, state=None))
    for name in ("x", "A", "state", "D"):
        with pytest.raises(RuntimeError, match="no gradient"):
            m2_amd.selective_scan_step(**dict(s, **{name: s[name].clone().requires_grad_()}))
    with torch.no_grad():
        m2_amd.selective_scan_step(**dict(s, x=s["x"].clone().requires_grad_()))
    # a state that a graph has kept and a step has moved on is noticed
    state = s["state"].clone()
    y = m2_amd.selective_scan(**dict(_scan_args(gpu), state=state, dt_bias=s["dt_bias"].clone().requires_grad_()))
    m2_amd.selective_scan_step(**dict(s, state=state))
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_transforms_and_tangents_are_refused(gpu):
    import m2_amd
    import torch.autograd.forward_ad as fwAD
    x = torch.randn(3, 2, 9, 16, device=gpu)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: m2_amd.group_norm(v, 4))(x)
    with pytest.raises(RuntimeError), fwAD.dual_level():
        m2_amd.group_norm(fwAD.make_dual(x[0], x[1]), 4)

    class Own(torch.Tensor):
        pass

    with pytest.raises(TypeError, match="plain"):
        m2_amd.group_norm(x[0].as_subclass(Own), 4)


def _all_calls(gpu):
    """{name: (inputs that ask for gradients, call -> outputs)}"""
    import m2_amd
    c, s = _conv_args(gpu), _scan_args(gpu)
    n = {"x": torch.randn(3, 5, 16, device=gpu), "weight": torch.randn(16, device=gpu), "bias": torch.randn(16, device=gpu)}
    t = {"x": torch.randn(30, 16, device=gpu), "weight": torch.randn(16, device=gpu), "bias": torch.randn(16, device=gpu)}
    return {"conv": (c, lambda i: list(m2_amd.causal_conv(**i, activation="silu", return_state=True))),
            "scan": (s, lambda i: list(m2_amd.selective_scan(**i, dt_softplus=True, return_state=True))),
            "norm": (n, lambda i: [m2_amd.group_norm(**i, groups=4, activation="gelu")]), "norm_tokens": (t, lambda i: [m2_amd.group_norm(**i, groups=4, activation="silu")])}


def _leaves(ins):
    return {k: v.detach().clone().requires_grad_() for k, v in ins.items()}


def _ones(outs):
    g = torch.Generator(device=outs[0].device).manual_seed(3)
    return [torch.randn(o.shape, generator=g, device=o.device).to(o.dtype) for o in outs]


@pytest.mark.parametrize("which", ["conv", "scan", "norm", "norm_tokens"])
def test_what_autograd_asks(gpu, which):
    """One input at a time, one output at a time, kept graphs, second derivatives, hooks on what is saved, in-place changes, gradients that are expanded."""
    ins, call = _all_calls(gpu)[which]
    leaves = _leaves(ins)
    outs = call(leaves)
    given = _ones(outs)
    whole = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), given, retain_graph=True)))
    again = torch.autograd.grad(outs, list(leaves.values()), given)
    assert all(torch.equal(a, b) for a, b in zip(whole.values(), again))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(outs, list(leaves.values()), given)
    for name in ins:
        alone = dict(ins)
        alone[name] = ins[name].detach().clone().requires_grad_()
        got, = torch.autograd.grad(call(alone), [alone[name]], given)
        assert torch.equal(got, whole[name]), name
    if len(outs) == 2:      # the gradient is the sum of those of either output
        parts = [torch.autograd.grad(call(leaves)[i], list(leaves.values()), given[i], allow_unused=True) for i in (0, 1)]
        for name, a, b in zip(leaves, *parts):
            both = sum(t.double() for t in (a, b) if t is not None)
            # two sums of the same terms, each off by 2^-24 of what it passes through: 2^-16 of the largest is far above
            assert (both - whole[name].double()).abs().max() <= 2.0 ** -16 * max(1.0, *(t.abs().max().item() for t in (a, b) if t is not None)), name
    v = _leaves(ins)
    g = torch.autograd.grad(call(v), list(v.values()), given, create_graph=True)
    assert torch.equal(g[0], whole[list(v)[0]])
    with pytest.raises(RuntimeError, match="second derivative"):
        g[0].sum().backward()
    for pack, unpack in ((lambda t: t.clone(), lambda t: t), (lambda t: t.cpu(), lambda t: t.to(gpu)), (lambda t: t, lambda t: torch.cat([t, t], -1)[..., :t.shape[-1]] if t.dim() else t)):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            v = _leaves(ins)
            outs = call(v)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(outs, list(v.values()), given), whole.values()))
    for unpack in (lambda t: t.double(), lambda t: t[..., :1], lambda t: t.cpu()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            v = _leaves(ins)
            outs = call(v)
        with pytest.raises(RuntimeError, match="came back"):
            torch.autograd.grad(outs, list(v.values()), given)
    v = _leaves(ins)
    outs = call(v)
    with torch.no_grad():
        v["x"].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(outs, list(v.values()), given)
    # a sum's gradient is one value expanded; broadcast inputs get the sum of their gradients
    v = _leaves(ins)
    a = torch.autograd.grad(sum(o.sum() for o in call(v)), list(v.values()))
    b = torch.autograd.grad(call(v), list(v.values()), [torch.ones_like(o) for o in given])
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    one = ins["x"][:1].clone().requires_grad_()
    wide = dict(ins, x=one.expand_as(ins["x"]))
    full = dict(ins, x=one.detach().expand_as(ins["x"]).contiguous().requires_grad_())
    p, = torch.autograd.grad(call(wide), [one], given)
    q, = torch.autograd.grad(call(full), [full["x"]], given)
    assert torch.equal(p, q.sum(0, keepdim=True))
    # one tensor as two inputs
    if which == "scan":
        v = _leaves(ins)
        p, = torch.autograd.grad(call(dict(v, dt=v["x"])), [v["x"]], given)
        u = _leaves(dict(ins, dt=ins["x"]))
        q = torch.autograd.grad(call(u), [u["x"], u["dt"]], given)
        assert torch.equal(p, q[0] + q[1])
    # views whose memory holds the negatives of their values
    negative = dict(ins, x=torch._neg_view(-ins["x"]))
    assert negative["x"].is_neg() and all(torch.equal(a, b) for a, b in zip(call(negative), call(ins)))


@pytest.mark.parametrize("which", ["conv", "scan", "norm", "norm_tokens"])
def test_streams_and_captured_graphs(gpu, which):
    """Two captured forward and backward passes, replayed in turns on two streams between eager calls, give what eager calls give."""
    ins, call = _all_calls(gpu)[which]
    sets = [{k: v * (1 + 0.1 * i) for k, v in ins.items()} for i in range(3)]
    given = _ones(call(ins))

    def run(i):
        v = {k: t.detach().requires_grad_() for k, t in i.items()}
        outs = call(v)
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, list(v.values()), given))

    want = [run(s) for s in sets]
    side = torch.cuda.Stream()
    graphs, outs, held = [], [], [{k: v.clone() for k, v in s.items()} for s in sets[:2]]
    for i in range(2):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(held[i])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(held[i]))
        graphs.append(graph)
    for turn in range(4):
        for i in range(2):
            for k, v in held[i].items():
                v.copy_(sets[(i + turn) % 3][k])
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        eager = run(sets[2])
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[(i + turn) % 3]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[2]))
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(run(sets[0]), want[0]))


@pytest.mark.parametrize("which", ["conv", "scan", "norm"])
def test_capture_beside_a_living_graph_is_refused(gpu, which):
    """A leaf that an eager graph of another stream holds: the capture's backward pass would leave its stream.  The forward is refused; once the graph is gone it is captured."""
    ins, call = _all_calls(gpu)[which]
    v = _leaves(ins)
    alive = call(v)
    graph = torch.cuda.CUDAGraph()
    refused = False
    with torch.cuda.graph(graph):
        try:
            call(v)
        except RuntimeError as e:
            refused = "stream capture" in str(e)
        call({k: t.detach() for k, t in v.items()})      # without gradients it is captured
    assert refused
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call(v)
        grads = torch.autograd.grad(outs, list(v.values()), [torch.ones_like(o) for o in outs])
    graph.replay()
    torch.cuda.synchronize()
    fresh = _leaves(ins)
    outs = call(fresh)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(outs, list(fresh.values()), [torch.ones_like(o) for o in outs])))


def test_steps_captured(gpu):
    """A token's step as one graph: replays move the states on in place."""
    import m2_amd
    c, s = _conv_args(gpu), {k: v[:, 0] if k in ("x", "dt", "B", "C", "z") else v for k, v in _scan_args(gpu).items()}
    conv_state, state = c["state"].clone(), s["state"].clone()

    def step(cs, ss):
        x = m2_amd.causal_conv_step(c["x"][:, 0], cs, c["weight"], c["bias"], "silu")
        x = m2_amd.group_norm(x, 4, activation="silu")
        return m2_amd.selective_scan_step(**dict(s, x=x, state=ss), dt_softplus=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(c["state"].clone(), s["state"].clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(conv_state, state)
    conv_state.copy_(c["state"])
    state.copy_(s["state"])
    eager = c["state"].clone(), s["state"].clone()
    for _ in range(5):
        graph.replay()
        want = step(*eager)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(conv_state, eager[0]) and torch.equal(state, eager[1])


def test_inference_mode(gpu):
    import m2_amd
    c = _conv_args(gpu)
    with torch.inference_mode():
        state = c["state"].clone()
        y = m2_amd.causal_conv_step(c["x"][:, 0], state, c["weight"])
        z = m2_amd.group_norm(y, 4)
    assert torch.equal(z, m2_amd.group_norm(m2_amd.causal_conv_step(c["x"][:, 0], c["state"].clone(), c["weight"]), 4))

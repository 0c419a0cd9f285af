"""GPU tests of how the prediction network's and the decoder's operators may be called: captured calls on leaves that the call
has to lay out, forward-mode derivatives, results that a compiled graph uses only through the caller's buffer, searches of
more frames than a history has tokens, gradients of some inputs, several graphs and threads."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from test_operator_calls import writers

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def apart(*shape):
    """A leaf whose elements are not adjacent, so that the call makes a copy of it."""
    t = torch.randn(*shape, 2, generator=torch.Generator().manual_seed(7)).to(DEV)
    return t[..., 0].requires_grad_(True)


def scan_args():
    r = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(8)).to(DEV)  # noqa: E731
    return dict(x=r(2, 5, 64), dt=r(2, 5, 64), A=-r(64, 8).abs(), B=r(2, 5, 8), C=r(2, 5, 8), D=r(64), z=r(2, 5, 64), dt_bias=r(64),
                initial_state=r(2, 64, 8))


def conv_args():
    r = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(9)).to(DEV)  # noqa: E731
    return dict(x=r(2, 5, 64), weight=r(64, 4), bias=r(64), initial_state=r(2, 3, 64))


@pytest.mark.parametrize("op,name", [("selective_scan", n) for n in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "initial_state")] +
                         [("causal_conv", n) for n in ("x", "weight", "bias", "initial_state")])
def test_capture_is_refused_for_a_leaf_that_the_call_lays_out(op, name):
    """Refused before anything is launched, as for a leaf that the call takes as it is."""
    import rnnt_amd

    args = scan_args() if op == "selective_scan" else conv_args()
    args[name] = apart(*args[name].shape)
    assert args[name].is_leaf and not args[name].is_contiguous()
    held = getattr(rnnt_amd, op)(**args)
    graph, scratch = torch.cuda.CUDAGraph(), torch.zeros(1, device=DEV)
    with torch.cuda.graph(graph):
        scratch.add_(1)
        with pytest.raises(RuntimeError, match="cannot be captured while"):
            getattr(rnnt_amd, op)(**args)
    del held


def test_a_forward_pass_is_captured_without_gradients_beside_an_eager_graph():
    """Under no_grad there is no backward pass in the capture, and nothing to refuse."""
    import rnnt_amd

    for op, args in (("selective_scan", scan_args()), ("causal_conv", conv_args())):
        leaves = {k: v.requires_grad_(True) for k, v in args.items()}
        held = getattr(rnnt_amd, op)(**leaves)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph), torch.no_grad():
            out = getattr(rnnt_amd, op)(**leaves)
        for seed in range(3):
            with torch.no_grad():
                args["x"].copy_(torch.randn(args["x"].shape, generator=torch.Generator().manual_seed(seed)))
                graph.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(p, q) for p, q in zip(out, getattr(rnnt_amd, op)(**leaves)))
        del held


def test_a_tangent_is_refused_on_the_device():
    import rnnt_amd

    for op, args in (("selective_scan", scan_args()), ("causal_conv", conv_args())):
        for name in args:
            with fwAD.dual_level():
                dual = fwAD.make_dual(args[name], torch.ones_like(args[name]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    getattr(rnnt_amd, op)(**{**args, name: dual})
            getattr(rnnt_amd, op)(**args)
    net = rnnt_amd.PredictionNet(12, 8, 8).to(DEV)
    name, weight = "embedding.weight", net.embedding.weight
    with fwAD.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.functional_call(net, {name: fwAD.make_dual(weight.detach(), torch.ones_like(weight))},
                                   (torch.zeros(1, 2, dtype=torch.int32, device=DEV),))


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
@pytest.mark.parametrize("fn,args,op", writers(), ids=lambda v: v if isinstance(v, str) else "")
def test_a_compiled_graph_writes_the_callers_buffer(fn, args, op):
    from rnnt_amd import _torch_binding

    _torch_binding.load()
    args = [t.to(DEV) for t in args]
    want = fn(*args[:-1], torch.zeros_like(args[-1]))
    assert torch.count_nonzero(want)
    out = torch.zeros_like(want)
    for graph in (torch.jit.script(fn), torch.jit.trace(fn, (*args[:-1], torch.zeros_like(want)), check_trace=False)):
        out.zero_()
        for _ in range(3):      # (the first runs of a compiled graph record it, the later ones are optimised)
            graph(*args[:-1], out)
        assert torch.equal(out, want)


def search_model(B, T, V=7, He=8, Hd=8):
    import rnnt_amd

    torch.manual_seed(11)
    net = rnnt_amd.PredictionNet(V, 8, Hd, layers=1).to(DEV).eval()
    joint = rnnt_amd.JointNet(He, 12, V, "sum").to(DEV).eval()
    return net, joint, torch.randn(B, T, He, generator=torch.Generator().manual_seed(12)).to(DEV)


def test_searches_of_more_frames_than_a_history_has_tokens():
    """Rules that look at no history do not limit the frames; penalties limit the emissions."""
    import rnnt_amd

    T, V = 65700, 7
    net, joint, enc = search_model(1, T)
    quiet = torch.zeros(V, device=DEV)
    quiet[0] = 100.0                                                 # blank at every frame
    mask = rnnt_amd.pack_allowed(torch.ones(V, dtype=torch.bool)).to(DEV)
    for rules in (rnnt_amd.LogitRules(bias=quiet), rnnt_amd.LogitRules(bias=quiet, allowed=mask),
                  rnnt_amd.LogitRules(bias=quiet, allowed=lambda tokens: mask), rnnt_amd.LogitRules(bias=quiet, presence_penalty=1.0)):
        assert rnnt_amd.greedy_decode(enc[0], T, net, joint, window=8192, rules=rules) == []
    assert rnnt_amd.greedy_search_batch(enc, net, joint, window=8192, rules=rnnt_amd.LogitRules(bias=quiet))[0] == [[]]


def test_neutral_penalties_give_what_a_counted_history_gives():
    """With a history given, tokens are counted; neutral penalties then leave every logit as it is, to the bit."""
    import rnnt_amd

    net, joint, enc = search_model(3, 60)
    bias = torch.randn(3, 7, generator=torch.Generator().manual_seed(13)).to(DEV)
    allowed = lambda tokens: rnnt_amd.pack_allowed(torch.arange(7) != (tokens[-1] if tokens else 3))  # noqa: E731
    history = torch.full((3, 1), 2, dtype=torch.int32, device=DEV)
    for rules in (dict(bias=bias), dict(allowed=allowed), dict(bias=bias[0], allowed=allowed), {}):
        free = rnnt_amd.greedy_search_batch(enc, net, joint, window=5, rules=rnnt_amd.LogitRules(**rules))
        counted = rnnt_amd.greedy_search_batch(enc, net, joint, window=5, rules=rnnt_amd.LogitRules(**rules, history=history))
        assert free[0] == counted[0] and torch.equal(free[1], counted[1])
        assert sum(map(len, free[0])) > 3
        one = {**rules, **({"bias": bias[:1]} if rules.get("bias") is bias else {})}
        free, counted = (rnnt_amd.greedy_decode(enc[0], 60, net, joint, window=5, rules=rnnt_amd.LogitRules(**one, **h))
                         for h in ({}, dict(history=history[:1])))
        assert free == counted and free


def embed_args():
    return dict(weight=torch.randn(12, 16, generator=torch.Generator().manual_seed(4)).to(DEV))


def all_ops():
    """name -> (call, tensors that have a gradient)."""
    import rnnt_amd

    tokens = torch.randint(0, 12, (3, 700), generator=torch.Generator().manual_seed(5)).to(DEV)
    return {"token_embedding": (lambda weight: (rnnt_amd.token_embedding(tokens, weight, 0.5, 3),), embed_args()),
            "causal_conv": (rnnt_amd.causal_conv, conv_args()), "selective_scan": (rnnt_amd.selective_scan, scan_args())}


def grads_of(call, args, names, create_graph=False):
    leaves = {k: v.detach().requires_grad_(k in names) for k, v in args.items()}
    outs = call(**leaves)
    gos = [torch.linspace(-1, 1, o.numel(), device=DEV).view(o.shape) for o in outs]
    return dict(zip(names, torch.autograd.grad(outs, [leaves[k] for k in names], gos, create_graph=create_graph)))


@pytest.mark.parametrize("op", ["token_embedding", "causal_conv", "selective_scan"])
def test_gradients_of_one_input_alone_and_of_required_arguments_only(op):
    """The same bits whichever inputs require grad; what is asked for with create_graph comes, and raises when differentiated again."""
    call, args = all_ops()[op]
    every = grads_of(call, args, list(args))
    for name in args:
        assert torch.equal(grads_of(call, args, [name])[name], every[name]), name
    required = {k: v for k, v in args.items() if k in ("weight", "x", "dt", "A", "B", "C")}
    plain, kept = (grads_of(call, required, list(required), create_graph=c) for c in (False, True))
    for name in required:
        assert torch.equal(plain[name], kept[name])
        with pytest.raises(RuntimeError, match="differentiated twice"):
            kept[name].sum().backward(retain_graph=True)


@pytest.mark.parametrize("op", ["causal_conv", "selective_scan"])
def test_an_input_changed_before_the_backward_pass_is_noticed(op):
    call, args = all_ops()[op]
    for name in args:
        if name == "initial_state" and op == "selective_scan":
            continue                                                 # (kept by the forward pass: nothing reads it again)
        leaves = {k: (v.detach().requires_grad_(True) * 1) for k, v in args.items()}
        total = call(**leaves)[0].sum()
        with torch.no_grad():
            leaves[name].add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            total.backward()


def test_two_captured_graphs_that_share_their_memory():
    """A training pass in each, one pool, replayed in turn with eager passes between: each is its own eager pass's result."""
    import rnnt_amd

    pool, graphs = None, []
    for L in (150, 33):
        a = {k: v.clone() for k, v in scan_args().items()}
        g = torch.Generator().manual_seed(L)
        for k, last in (("x", 64), ("dt", 64), ("B", 8), ("C", 8), ("z", 64)):
            a[k] = torch.randn(2, L, last, generator=g).to(DEV)
        leaves = {k: v.requires_grad_(True) for k, v in a.items()}
        gy = torch.randn(2, L, 64, generator=g).to(DEV)

        def fn(leaves=leaves, gy=gy):
            y, _ = rnnt_amd.selective_scan(**leaves)
            return (y.detach(), *torch.autograd.grad(y, list(leaves.values()), gy))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = fn()
        pool = graph.pool()
        graphs.append((graph, out, fn, leaves))
    for seed in range(3):
        for graph, out, fn, leaves in graphs:
            with torch.no_grad():
                leaves["x"].copy_(torch.randn(leaves["x"].shape, generator=torch.Generator().manual_seed(seed)))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, fn()))


def test_two_threads_each_on_its_stream():
    """Nothing is shared between calls: the same bits as alone."""
    import threading

    jobs = list(all_ops().values())[1:]
    alone = [grads_of(call, args, list(args)) for call, args in jobs]
    torch.cuda.synchronize()
    errors = []

    def work(call, args, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = grads_of(call, args, list(args))
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(got[k], want[k]) for k in want)
        except BaseException as e:  # noqa: B902
            errors.append(e)

    threads = [threading.Thread(target=work, args=(*job, want)) for job, want in zip(jobs * 2, alone * 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_a_recomputed_layer_gives_the_same_gradients():
    import rnnt_amd
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(2)
    net = rnnt_amd.PredictionNet(12, 16, 8, layers=2).to(DEV)
    tokens = torch.randint(0, 12, (3, 40), generator=torch.Generator().manual_seed(6)).to(DEV)
    grads = []
    for again in (False, True):
        net.zero_grad()
        u = net.embedding(tokens)
        for layer in net.layers:
            u = checkpoint(lambda v, f=layer: f(v, None, None, None)[0], u, use_reentrant=False) if again else layer(u, None, None, None)[0]
        u.square().sum().backward()
        grads.append({k: p.grad.clone() for k, p in net.named_parameters() if p.grad is not None})
    assert grads[0].keys() == grads[1].keys() and all(torch.equal(grads[0][k], grads[1][k]) for k in grads[0])

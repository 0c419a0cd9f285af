"""GPU tests of how the prediction network's and the decoder's operators may be called: captured calls on leaves that the call
has to lay out, forward-mode derivatives, results that a compiled graph uses only through the caller's buffer."""
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

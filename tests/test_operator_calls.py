"""CPU tests of how the prediction network's and the decoder's operators may be called.  Nothing is launched."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import rnnt_amd

R = rnnt_amd.LogitRules


def calls():
    """name -> (call of keyword tensors, the tensors)."""
    r = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(3))  # noqa: E731
    scan = dict(x=r(2, 5, 6), dt=r(2, 5, 6), A=-r(6, 8).abs(), B=r(2, 5, 8), C=r(2, 5, 8), D=r(6), z=r(2, 5, 6), dt_bias=r(6),
                initial_state=r(2, 6, 8))
    step = {k: v[:, 0] if k in ("x", "dt", "B", "C", "z") else v for k, v in scan.items() if k != "initial_state"}
    rules = dict(x=r(4, 9), bias=r(9))
    return {
        "token_embedding": (lambda weight: rnnt_amd.token_embedding(torch.zeros(3, dtype=torch.int32), weight), dict(weight=r(5, 4))),
        "causal_conv": (rnnt_amd.causal_conv, dict(x=r(2, 5, 6), weight=r(6, 4), bias=r(6), initial_state=r(2, 3, 6))),
        "causal_conv_step": (rnnt_amd.causal_conv_step, dict(x=r(2, 6), state=r(2, 3, 6), weight=r(6, 4), bias=r(6))),
        "selective_scan": (rnnt_amd.selective_scan, scan),
        "selective_scan_step": (rnnt_amd.selective_scan_step, {**step, "state": r(2, 6, 8)}),
        "row_max_logp": (lambda x, bias: rnnt_amd.row_max_logp(x, R(bias=bias)), rules),
        "process_logits": (lambda x, bias: rnnt_amd.process_logits(x, R(bias=bias)), rules),
        "row_argmax": (lambda x, bias: rnnt_amd.row_argmax(x, R(bias=bias)), rules),
    }


@pytest.mark.parametrize("op,name", [(op, k) for op, (_, t) in calls().items() for k in t])
def test_a_tangent_is_refused_and_not_lost(op, name):
    """Whether or not the input requires grad, and without grad mode too (which leaves forward derivatives on); a token alone has no
    derivative, so that row_argmax goes on to the next check."""
    call, tensors = calls()[op]
    for requires_grad in (False, True):
        for mode in (torch.enable_grad(), torch.no_grad()):
            with fwAD.dual_level(), mode:
                leaf = tensors[name].clone().requires_grad_(requires_grad)
                dual = fwAD.make_dual(leaf, torch.ones_like(leaf))
                if op == "row_argmax":
                    with pytest.raises(RuntimeError, match="no CPU path"):
                        call(**{**tensors, name: dual})
                    continue
                with pytest.raises(NotImplementedError, match=op + " has no forward-mode derivative"):
                    call(**{**tensors, name: dual})
    with pytest.raises(RuntimeError, match="no CPU path"):       # outside of a level, nothing is refused for it
        call(**tensors)


def write_logits(x: torch.Tensor, out: torch.Tensor):
    torch.ops.rnnt_amd.process_logits(x, None, None, None, None, 1.0, 0.0, 0.0, out)
    return out


def write_conv(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, out: torch.Tensor):
    torch.ops.rnnt_amd.causal_conv_step(x, state, weight, None, True, out)
    return out


def write_scan(x: torch.Tensor, A: torch.Tensor, B: torch.Tensor, state: torch.Tensor, out: torch.Tensor):
    torch.ops.rnnt_amd.selective_scan_step(x, x, A, B, B, state, None, None, None, out)
    return out


def writers():
    """(function that writes the last of its tensors and uses nothing that the call returns, its tensors, name of the operator)"""
    r = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(5))  # noqa: E731
    return [(write_logits, [r(3, 9), torch.zeros(3, 9)], "process_logits"),
            (write_conv, [r(2, 6), r(2, 3, 6), r(6, 4), torch.zeros(2, 3, 6)], "causal_conv_step"),
            (write_scan, [r(2, 6), -r(6, 8).abs(), r(2, 8), r(2, 6, 8), torch.zeros(2, 6, 8)], "selective_scan_step")]


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
@pytest.mark.parametrize("fn,args,op", writers(), ids=lambda v: v if isinstance(v, str) else "")
def test_a_compiled_graph_keeps_a_call_for_the_buffer_it_writes(fn, args, op):
    from rnnt_amd import _torch_binding

    schema = getattr(_torch_binding.load(), op).default._schema
    assert schema.is_mutable
    assert [a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write] == [
        "out" if op == "process_logits" else "state_out"]
    script = torch.jit.script(fn)
    graph = script.graph.copy()
    torch._C._jit_pass_dce(graph)
    assert "rnnt_amd::" + op in str(graph)
    with pytest.raises(RuntimeError, match="no CPU path"):
        script(*args)


def test_calls_that_write_no_buffer_say_so():
    from rnnt_amd import _torch_binding

    ops = _torch_binding.load()
    for name in ("token_embedding", "causal_conv", "selective_scan", "row_rules"):
        assert not getattr(ops, name).default._schema.is_mutable


@pytest.mark.parametrize("fn,args,op", writers(), ids=lambda v: v if isinstance(v, str) else "")
def test_a_buffer_that_autograd_follows_is_refused(fn, args, op):
    """Overwritten, it would keep the gradient of the values that are gone; under no_grad it is written, as torch's own calls do."""
    from rnnt_amd import _torch_binding

    _torch_binding.load()
    leaf = args[-1].requires_grad_(True)
    for out in (leaf, leaf * 1):
        with pytest.raises(RuntimeError, match=op + " is for decoding and has no backward"):
            fn(*args[:-1], out)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            fn(*args[:-1], out)
    with fwAD.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
        fn(*args[:-1], fwAD.make_dual(leaf.detach(), torch.ones_like(leaf)))


@pytest.mark.parametrize("op", ["row_max_logp", "process_logits", "row_argmax"])
@pytest.mark.parametrize("name", ["x", "bias"])
def test_values_without_a_backward_are_refused_where_a_gradient_is_asked_for(op, name):
    """One answer from both calls that give values; a token has no derivative."""
    call, tensors = calls()[op]
    args = {**tensors, name: tensors[name].requires_grad_(True)}
    with pytest.raises(RuntimeError, match="no CPU path" if op == "row_argmax" else op + " is for decoding and has no backward"):
        call(**args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
        call(**args)


def test_search_rules_keep_a_history_only_where_a_penalty_looks_at_it():
    from rnnt_amd.rules import HistoryRules

    frames = 70000                                                   # more than 16 bits count
    words = torch.tensor([7], dtype=torch.int32)
    said = []
    kept = HistoryRules(R(bias=torch.ones(2, 9), allowed=lambda tokens: said.append(tokens) or words), 2, 9, frames, "cpu")
    kept.emit([1], [4])
    assert said == [[], [], [4]]                                     # a callable mask still follows what is emitted
    now = kept.of([1])
    assert now.history is None and now.bias.tolist() == [[1.0] * 9] and now.allowed.tolist() == [[7]]
    kept.tokens[0] = [1] * 65535
    kept.emit([0], [1])                                              # nothing is counted: no limit
    for penalty in (dict(repetition_penalty=2.0), dict(presence_penalty=-1.0), dict(frequency_penalty=0.5)):
        kept = HistoryRules(R(**penalty), 2, 9, frames, "cpu")
        kept.emit([0, 1], [4, 5])
        kept.emit([1], [6])
        assert kept.of([0, 1]).history.tolist() == [[4, -1], [5, 6]]
        kept.tokens[0] = [1] * 65534
        kept.emit([0], [3])                                          # the last one that can be counted
        assert kept.of([0]).history.shape == (1, 65535) and int(kept.of([0]).history[0, -1]) == 3
        with pytest.raises(ValueError, match="longer than 65535"):
            kept.emit([0], [3])
    assert HistoryRules(R(presence_penalty=1.0), 2, 9, 5, "cpu").history.shape == (2, 5)

"""CPU tests: what the prediction network's and the decoder's operators refuse, the plain forms that the GPU tests check
against (their own gradients, by differences), and the C entry points' checks.  Nothing is launched."""
import ctypes

import pytest
import torch

import rnnt_amd
from rnnt_amd import _lib

import plain_operators as plain

F32, I32 = torch.float32, torch.int32


def scan_inputs(B=2, L=5, D=6, N=8, dtype=F32):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    return dict(x=r(B, L, D), dt=r(B, L, D), A=-torch.rand(D, N, generator=g), B=r(B, L, N), C=r(B, L, N))


def test_cpu_tensors_raise_after_the_shape_checks():
    a = scan_inputs()
    w = torch.zeros(6, 4)
    calls = [
        lambda: rnnt_amd.token_embedding(torch.zeros(3, dtype=I32), torch.zeros(5, 4)),
        lambda: rnnt_amd.causal_conv(a["x"], w),
        lambda: rnnt_amd.causal_conv_step(a["x"][:, 0], torch.zeros(2, 3, 6), w),
        lambda: rnnt_amd.selective_scan(**a),
        lambda: rnnt_amd.selective_scan_step(a["x"][:, 0], a["dt"][:, 0], a["A"], a["B"][:, 0], a["C"][:, 0], torch.zeros(2, 6, 8)),
        lambda: rnnt_amd.row_argmax(torch.zeros(2, 5), rnnt_amd.LogitRules()),
        lambda: rnnt_amd.row_max_logp(torch.zeros(2, 5), rnnt_amd.LogitRules()),
        lambda: rnnt_amd.process_logits(torch.zeros(2, 5), rnnt_amd.LogitRules()),
    ]
    for call in calls:
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_embedding_refusals():
    f, w, t = rnnt_amd.token_embedding, torch.zeros(5, 4), torch.zeros(3, dtype=I32)
    with pytest.raises(TypeError, match="tokens must be"):
        f(t.float(), w)
    with pytest.raises(TypeError, match="weight must be"):
        f(t, w.double())
    with pytest.raises(ValueError, match="non-empty"):
        f(t, w[0:0])
    with pytest.raises(ValueError, match="non-empty"):
        f(t, torch.zeros(4))
    with pytest.raises(ValueError, match="tokens must not be empty"):
        f(t[:0], w)
    for padding in (5, -1):
        with pytest.raises(ValueError, match="padding_idx"):
            f(t, w, padding_idx=padding)
    for scale in (float("inf"), float("nan"), 1e300):
        with pytest.raises(ValueError, match="scale"):
            f(t, w, scale=scale)


def test_conv_refusals():
    f, x, w = rnnt_amd.causal_conv, torch.zeros(2, 5, 6), torch.zeros(6, 4)
    with pytest.raises(TypeError, match="x must be"):
        f(x.double(), w)
    with pytest.raises(ValueError, match="batch, length, dim"):
        f(x[0], w)
    with pytest.raises(ValueError, match="non-empty"):
        f(x[:, :0], w)
    for bad in (torch.zeros(6, 5), torch.zeros(6, 1), torch.zeros(5, 4), torch.zeros(6)):
        with pytest.raises(ValueError, match="weight must be"):
            f(x, bad)
    with pytest.raises(TypeError, match="weight must be torch.float32"):
        f(x, w.half())
    with pytest.raises(ValueError, match="bias must have shape"):
        f(x, w, torch.zeros(5))
    with pytest.raises(ValueError, match="initial_state must be"):
        f(x, w, initial_state=torch.zeros(2, 4, 6))
    with pytest.raises(TypeError, match="initial_state must have x's type"):
        f(x, w, initial_state=torch.zeros(2, 3, 6).half())
    with pytest.raises(TypeError, match="lengths must be torch.int32"):
        f(x, w, lengths=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="lengths must be a contiguous"):
        f(x, w, lengths=torch.zeros(3, dtype=I32))
    with pytest.raises(ValueError, match="activation"):
        f(x, w, activation="relu")
    with pytest.raises(ValueError, match="state must be"):
        rnnt_amd.causal_conv_step(x[:, 0], torch.zeros(2, 2, 6), w)
    with pytest.raises(ValueError, match="batch, dim"):
        rnnt_amd.causal_conv_step(x, torch.zeros(2, 3, 6), w)


def test_scan_refusals():
    f = rnnt_amd.selective_scan

    def call(**change):
        return f(**{**scan_inputs(), **change})

    a = scan_inputs()
    with pytest.raises(TypeError, match="x must be"):
        call(x=a["x"].double())
    with pytest.raises(ValueError, match="batch, length, dim"):
        call(x=a["x"][0])
    with pytest.raises(ValueError, match="8, 16 or 32 states"):
        call(A=torch.zeros(6, 12))
    with pytest.raises(ValueError, match="8, 16 or 32 states"):
        call(A=torch.zeros(5, 8))
    with pytest.raises(TypeError, match="A must be torch.float32"):
        call(A=a["A"].half())
    with pytest.raises(TypeError, match="dt must have x's type"):
        call(dt=a["dt"].half())
    with pytest.raises(ValueError, match="dt must agree"):
        call(dt=a["dt"][:, :4])
    with pytest.raises(ValueError, match="B must agree"):
        call(B=torch.zeros(2, 5, 16))
    with pytest.raises(ValueError, match="C must agree"):
        call(C=torch.zeros(1, 5, 8))
    with pytest.raises(ValueError, match="D must have shape"):
        call(D=torch.zeros(5))
    with pytest.raises(TypeError, match="dt_bias must be torch.float32"):
        call(dt_bias=torch.zeros(6).bfloat16())
    with pytest.raises(ValueError, match="z must agree"):
        call(z=torch.zeros(2, 5, 5))
    with pytest.raises(ValueError, match="initial_state must have shape"):
        call(initial_state=torch.zeros(2, 6, 16))
    with pytest.raises(TypeError, match="initial_state must be torch.float32"):
        call(initial_state=torch.zeros(2, 6, 8).half())
    with pytest.raises(ValueError, match="lengths must be a contiguous"):
        call(lengths=torch.zeros(4, dtype=I32)[::2])
    with pytest.raises(ValueError, match="state must have shape"):
        rnnt_amd.selective_scan_step(a["x"][:, 0], a["dt"][:, 0], a["A"], a["B"][:, 0], a["C"][:, 0], torch.zeros(1, 6, 8))


def test_rules_refusals():
    x, R = torch.zeros(6, 40), rnnt_amd.LogitRules

    def call(r, x=x):
        return rnnt_amd.process_logits(x, r)

    with pytest.raises(TypeError, match="LogitRules"):
        rnnt_amd.row_argmax(x, dict(bias=None))
    with pytest.raises(ValueError, match="rows, V"):
        call(R(), x[0])
    with pytest.raises(TypeError, match="x must be"):
        call(R(), x.double())
    with pytest.raises(TypeError, match="bias must be torch.float32"):
        call(R(bias=torch.zeros(40).half()))
    with pytest.raises(ValueError, match="bias must be"):
        call(R(bias=torch.zeros(41)))
    with pytest.raises(TypeError, match="one bit per token"):
        call(R(allowed=torch.ones(40, dtype=torch.bool)))
    with pytest.raises(ValueError, match="allowed must be"):
        call(R(allowed=torch.zeros(1, dtype=I32)))
    with pytest.raises(TypeError, match="history must be torch.int32"):
        call(R(history=torch.zeros(2, 3, dtype=torch.int64)))
    with pytest.raises(ValueError, match="history must be"):
        call(R(history=torch.zeros(3, dtype=I32)))
    with pytest.raises(ValueError, match="at most 65535"):
        call(R(history=torch.zeros(1, 65536, dtype=I32)))
    with pytest.raises(ValueError, match="history_lens needs history"):
        call(R(history_lens=torch.zeros(1, dtype=I32)))
    with pytest.raises(ValueError, match="history_lens must be"):
        call(R(history=torch.zeros(2, 3, dtype=I32), history_lens=torch.zeros(3, dtype=I32)))
    with pytest.raises(ValueError, match="contexts"):
        call(R(history=torch.zeros(2, 3, dtype=I32), bias=torch.zeros(3, 40)))
    with pytest.raises(ValueError, match="multiple of the contexts"):
        call(R(bias=torch.zeros(4, 40)))
    for bad in (0.0, -1.0, float("nan"), float("inf"), 1e-60):
        with pytest.raises(ValueError, match="repetition_penalty"):
            call(R(repetition_penalty=bad))
    with pytest.raises(ValueError, match="must be finite"):
        call(R(presence_penalty=float("nan")))
    with pytest.raises(ValueError, match="must be finite"):
        call(R(frequency_penalty=float("inf")))
    with pytest.raises(TypeError, match="callable"):
        call(R(allowed=lambda tokens: None))
    with pytest.raises(ValueError, match="torch.bool"):
        rnnt_amd.pack_allowed(torch.ones(3))


def test_pack_allowed():
    mask = torch.zeros(2, 70, dtype=torch.bool)
    mask[0, [0, 31, 32, 69]] = True
    mask[1, 33:] = True
    words = rnnt_amd.pack_allowed(mask)
    assert words.dtype is I32 and words.shape == (2, 3)
    back = torch.stack([(words[:, v // 32].long() >> (v % 32)) & 1 for v in range(70)], 1).bool()
    assert torch.equal(back, mask)
    assert rnnt_amd.pack_allowed(torch.ones(32, dtype=torch.bool)).tolist() == [-1]


def test_prediction_net_refusals_and_parameters():
    with pytest.raises(ValueError, match="state_size"):
        rnnt_amd.PredictionNet(10, 8, 8, state_size=12)
    with pytest.raises(ValueError, match="conv_width"):
        rnnt_amd.PredictionNet(10, 8, 8, conv_width=5)
    with pytest.raises(ValueError, match="layers"):
        rnnt_amd.PredictionNet(10, 8, 8, layers=0)
    net = rnnt_amd.PredictionNet(10, 8, 5)
    assert torch.count_nonzero(net.embedding.weight[0]) == 0
    with pytest.raises(ValueError, match=r"\[B, U\]"):
        net(torch.zeros(3, dtype=I32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        net(torch.zeros(2, 3, dtype=I32))


def test_c_entry_points_refuse_before_any_launch():
    lib = _lib.load()
    n = ctypes.c_size_t(0)
    one = ctypes.c_void_p(16)      # never read: every call below is refused for another argument
    assert lib.rnnt_token_embedding_forward(None, 0, 3, one, 4, 5, 4, 1.0, 0, one, None) == 2
    assert lib.rnnt_token_embedding_forward(one, 0, 0, one, 4, 5, 4, 1.0, 0, one, None) == 2
    assert lib.rnnt_token_embedding_forward(one, 0, 3, one, 3, 5, 4, 1.0, 0, one, None) == 2       # rows overlap
    assert lib.rnnt_token_embedding_forward(one, 0, 3, one, 4, 5, 4, 1.0, 7, one, None) == 2       # no such type
    assert lib.rnnt_token_embedding_workspace_size(0, 5, 4, ctypes.byref(n)) == 2
    assert lib.rnnt_token_embedding_workspace_size(3, 5, 4, None) == 2
    assert lib.rnnt_token_embedding_workspace_size(3, 5, 4, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.rnnt_token_embedding_workspace_size(3000, 5, 4, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.rnnt_token_embedding_backward(one, 0, 3, one, 4, 5, 4, 1.0, -1, 0, None, None, None) == 2
    assert lib.rnnt_token_embedding_backward(one, 0, 3000, one, 4, 5, 4, 1.0, -1, 0, one, None, None) == 2
    assert lib.rnnt_token_embedding_backward(one, 0, 3000, one, 4, 5, 4, 1.0, -1, 0, one, ctypes.c_void_p(8), None) == 2

    assert lib.rnnt_row_rules(one, 4, 8, 0, None, one, None, None, None) == 2
    rules = _lib.RnntRules(contexts=3, repetition_penalty=1.0)
    assert lib.rnnt_row_rules(one, 4, 8, 0, ctypes.byref(rules), one, None, None, None) == 2             # 4 rows of 3 contexts
    rules = _lib.RnntRules(contexts=1, repetition_penalty=1.0)
    assert lib.rnnt_row_rules(one, 4, 70001, 0, ctypes.byref(rules), one, None, None, None) == 2   # needs its workspace
    assert lib.rnnt_row_rules_workspace_size(4, 5455, 1, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.rnnt_row_rules_workspace_size(4, 70001, 1, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.rnnt_row_rules_workspace_size(4, 70001, 3, ctypes.byref(n)) == 2
    for change in (dict(history=16, history_stride=0), dict(history=16, history_stride=65536), dict(bias=16, bias_stride=7),
                   dict(allowed=16, allowed_stride=0, repetition_penalty=0.0), dict(repetition_penalty=float("nan")),
                   dict(presence_penalty=float("nan")), dict(contexts=0)):
        rules = _lib.RnntRules(**{**dict(contexts=2, repetition_penalty=1.0), **change})
        assert lib.rnnt_process_logits(one, 4, 8, 0, ctypes.byref(rules), one, None) == 2, change

    conv = dict(batch=2, length=3, dim=4, width=4, x=16, weight=16, y=16, initial_state=16, final_state=16, grad_y=16, grad_x=16,
                grad_weight=16, workspace=16)
    for fn, change in ((lib.rnnt_causal_conv_forward, dict(width=5)), (lib.rnnt_causal_conv_forward, dict(x=None)),
                       (lib.rnnt_causal_conv_forward, dict(length=0)), (lib.rnnt_causal_conv_forward, dict(dtype=9)),
                       (lib.rnnt_causal_conv_backward, dict(workspace=None)), (lib.rnnt_causal_conv_backward, dict(workspace=8)),
                       (lib.rnnt_causal_conv_step, dict(initial_state=None)), (lib.rnnt_causal_conv_step, dict(final_state=None))):
        assert fn(ctypes.byref(_lib.RnntConv(**{**conv, **change}))) == 2, change
    assert lib.rnnt_causal_conv_forward(None) == 2
    assert lib.rnnt_causal_conv_workspace_size(2, 3, 4, 5, ctypes.byref(n)) == 2

    scan = dict(batch=2, length=3, dim=4, state=16, x=16, dt=16, A=16, B=16, C=16, y=16, initial_state=16, final_state=16,
                chunk_states=16, grad_y=16, grad_x=16, grad_dt=16, grad_A=16, grad_B=16, grad_C=16, workspace=16)
    for fn, change in ((lib.rnnt_selective_scan_forward, dict(state=12)), (lib.rnnt_selective_scan_forward, dict(A=None)),
                       (lib.rnnt_selective_scan_forward, dict(chunk_states=8)), (lib.rnnt_selective_scan_forward, dict(workspace=None)), (lib.rnnt_selective_scan_forward, dict(dtype=-1)),
                       (lib.rnnt_selective_scan_backward, dict(chunk_states=None)), (lib.rnnt_selective_scan_backward, dict(z=16)),
                       (lib.rnnt_selective_scan_backward, dict(workspace=None)), (lib.rnnt_selective_scan_step, dict(final_state=None)),
                       (lib.rnnt_selective_scan_step, dict(initial_state=None))):
        assert fn(ctypes.byref(_lib.RnntScan(**{**scan, **change}))) == 2, change
    assert lib.rnnt_selective_scan_states_size(2, 33, 5, 16, ctypes.byref(n)) == 0
    assert n.value == (2 * 3 * 5 * 16 + (2 * 48 + 1) * 2 * 16) * 4   # states before steps 0, 16, 32; rows of B and C
    assert lib.rnnt_selective_scan_states_size(1 << 20, 1 << 20, 64, 16, ctypes.byref(n)) == 2


def test_structures_mirror_the_header():
    """Field names and kinds of the ctypes structures, in the header's order."""
    import os
    import re

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "rnnt_mi355.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, mirror in (("rnntRules", _lib.RnntRules), ("rnntConv", _lib.RnntConv), ("rnntScan", _lib.RnntScan)):
        end = text.index("} %s;" % name)
        body = text[text.rindex("typedef struct {", 0, end) + len("typedef struct {"):end]
        fields = []
        for line in body.split(";"):
            line = line.strip()
            if not line:
                continue
            kind = {"int": ctypes.c_int, "float": ctypes.c_float, "long long": ctypes.c_longlong}
            base = re.match(r"(?:const )?(long long|int|float|void)", line).group(0)
            for item in line[len(base):].split(","):
                item = item.strip()
                pointer = item.startswith("*")
                fields.append((item.lstrip("* "), ctypes.c_void_p if pointer else kind[base.replace("const ", "")]))
        assert fields == list(mirror._fields_), name


# ---- the plain forms' own gradients, by differences ---------------------------------------------------------------------
def _directional(fn, inputs, grads, outputs_grad):
    """<gradient, direction> against the central difference of <outputs, outputs_grad>, in 64 bits."""
    g = torch.Generator().manual_seed(11)
    for name in grads:
        v = torch.randn(inputs[name].shape, generator=g, dtype=torch.float64)
        e = 1e-6
        up, down = ({**inputs, name: inputs[name] + s * e * v} for s in (1, -1))
        total = lambda o: sum(float((o[k] * outputs_grad[k]).sum()) for k in outputs_grad)  # noqa: E731
        want = (total(fn(up)) - total(fn(down))) / (2 * e)
        got = float((grads[name] * v).sum())
        # central difference: error O(e^2) of the third derivative and 2^-53 / e of the values
        assert got == pytest.approx(want, rel=1e-6, abs=1e-6), name


def test_plain_scan_gradient_against_differences():
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    a = dict(x=r(2, 7, 3), dt=r(2, 7, 3), A=-torch.rand(3, 8, generator=g).double(), B=r(2, 7, 8), C=r(2, 7, 8), D=r(3), z=r(2, 7, 3),
             bias=r(3), init=r(2, 3, 8))
    lens, gy, gf = [7, 4], r(2, 7, 3), r(2, 3, 8)
    o = plain.scan(**a, lens=lens, gy=gy, gfinal=gf)
    live = (torch.arange(7)[None] < torch.tensor(lens)[:, None]).double()[..., None]
    _directional(lambda i: plain.scan(**i, lens=lens), a, {k: o["d" + k] for k in a}, dict(y=gy * live, state=gf))


def test_plain_conv_gradient_against_differences():
    g = torch.Generator().manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    a = dict(x=r(3, 6, 4), w=r(4, 4), b=r(4), init=r(3, 3, 4))
    lens, gy, gf = [6, 1, 0], r(3, 6, 4), r(3, 3, 4)
    for silu in (True, False):
        o = plain.conv(a["x"], a["w"], a["b"], a["init"], lens, silu, gy, gf)
        live = (torch.arange(6)[None] < torch.tensor(lens)[:, None]).double()[..., None]
        _directional(lambda i: plain.conv(i["x"], i["w"], i["b"], i["init"], lens, silu), a, {k: o["d" + k] for k in a},
                     dict(y=gy * live, state=gf))


def test_calls_beyond_a_launch_are_refused():
    """A launch has less than 2^32 threads, and positions are added in 32 bits."""
    one = torch.zeros(1, 1)
    with pytest.raises(ValueError, match="too many tokens"):
        rnnt_amd.token_embedding(torch.zeros(1, dtype=I32).expand((1 << 30) + 1), one)
    with pytest.raises(ValueError, match="too large a weight"):
        rnnt_amd.token_embedding(torch.zeros(1, dtype=I32), one.expand((1 << 26) + 1, 1))
    with pytest.raises(ValueError, match="too large a weight"):
        rnnt_amd.token_embedding(torch.zeros(1, dtype=I32), one.expand(1, (1 << 21) + 1))
    for rows, V in ((1 << 22, 1), (1 << 18, 70001 * 2)):
        with pytest.raises(ValueError, match="too many rows"):
            rnnt_amd.row_argmax(one.expand(rows, V), rnnt_amd.LogitRules())
    for B, L, D in ((1 << 24, 1, 64), (1, 1 << 27, 1), (4, 1, 1 << 25)):
        x = one.expand(B, L, D)
        bc = one.expand(B, L, 16)
        with pytest.raises(ValueError, match="too large for one call"):
            rnnt_amd.selective_scan(x, x, one.expand(D, 16), bc, bc)
    for B, L, D in ((1 << 27, 1, 1), (1, 1, 1 << 25)):
        with pytest.raises(ValueError, match="too large for one call"):
            rnnt_amd.causal_conv(one.expand(B, L, D), one.expand(D, 4))


def test_search_rules_are_checked():
    from rnnt_amd.rules import HistoryRules

    R = rnnt_amd.LogitRules
    history, lens = torch.tensor([[3, 4], [5, 6]], dtype=I32), torch.tensor([2, 1], dtype=I32)
    kept = HistoryRules(R(history=history, history_lens=lens), 2, 9, 4, "cpu")
    kept.emit([1], [7])
    assert kept.of([0, 1]).history.tolist() == [[3, 4, -1], [5, -1, 7]]
    for bad, error in ((R(history=history.long()), TypeError), (R(history=history, history_lens=lens.long()), TypeError),
                       (R(history=history, history_lens=lens[:1]), ValueError), (R(history_lens=lens), ValueError),
                       (R(history=history[:1]), ValueError), (R(bias=torch.zeros(8)), ValueError),
                       (R(allowed=lambda tokens: torch.zeros(2, dtype=I32)), ValueError), (R(history=history), None)):
        if error is None:
            with pytest.raises(ValueError, match="longer than 65535"):
                HistoryRules(bad, 2, 9, 65534, "cpu")
            continue
        with pytest.raises(error):
            HistoryRules(bad, 2, 9, 4, "cpu")

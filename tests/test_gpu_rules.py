"""GPU tests of decoding rules: process_logits bit for bit against the fp32 formula, row_argmax / row_max_logp on its
result, and the greedy searches under rules and over a PredictionNet against loops written out here."""
import math

import pytest
import torch

import plain_operators as plain

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = plain.U


def make(contexts, window, V, hist, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(contexts * window, V, generator=g) * spread).to(dtype)
    return x, dict(bias=torch.randn(contexts, V, generator=g) * (torch.rand(contexts, V, generator=g) < 0.2),
                   allowed=torch.rand(contexts, V, generator=g) < 0.8,
                   history=torch.randint(0, V, (contexts, hist), generator=g, dtype=torch.int32),
                   history_lens=torch.randint(0, hist + 1, (contexts,), generator=g, dtype=torch.int32),
                   repetition=1.3, presence=0.4, frequency=0.15)


def rules_of(r):
    import rnnt_amd

    dev = lambda k: r[k].to(DEV) if r.get(k) is not None else None  # noqa: E731
    return rnnt_amd.LogitRules(bias=dev("bias"), allowed=None if r.get("allowed") is None else rnnt_amd.pack_allowed(r["allowed"]).to(DEV),
                               history=dev("history"), history_lens=dev("history_lens"), repetition_penalty=r.get("repetition", 1.0),
                               presence_penalty=r.get("presence", 0.0), frequency_penalty=r.get("frequency", 0.0))


def check(x, r):
    import rnnt_amd

    want = plain.rules32(x, x.shape[1], **r)
    rules, xd = rules_of(r), x.to(DEV)
    got = rnnt_amd.process_logits(xd, rules)
    assert got.dtype is x.dtype
    same = got.cpu().float().nan_to_num(nan=7.7e33) == want.to(x.dtype).float().nan_to_num(nan=7.7e33)
    assert bool(same.all()), (got.cpu()[~same][:5], want[~same][:5])
    token, logp = rnnt_amd.row_max_logp(xd, rules)
    assert torch.equal(token, rnnt_amd.row_argmax(xd, rules))
    first = torch.argmax(want, dim=1)                       # (NaN counts as the maximum, the first index wins)
    assert torch.equal(token.cpu().long(), first)
    w = want.double()
    # (x - max first: at the type's lowest value max - logsumexp would lose the logarithm even in 64 bits)
    ref = -torch.log(torch.exp(w - w.gather(1, first[:, None])).sum(1))
    plain.assert_within(logp, ref.where(torch.isfinite(w.amax(1)), torch.full_like(ref, math.nan)),
                        # n / 256 additions in a lane, 16 joins; an exponent x - m is off by 2 |x - m| u and counts at most 1 / e of it
                        (48 + x.shape[1] / 256) * U + 2 * U * ref.abs(), "logp")
    out = xd.clone()
    assert rnnt_amd.process_logits(out, rules, out=out).data_ptr() == out.data_ptr() and torch.equal(out.isnan(), got.isnan())
    assert torch.equal(out.nan_to_num(), got.nan_to_num())


@pytest.mark.parametrize("dtype", plain.TYPES)
@pytest.mark.parametrize("contexts,window,V,hist", [(1, 1, 1, 1), (2, 3, 7, 5), (1, 1, 33, 40), (3, 2, 64, 9), (2, 2, 4232, 60), (1, 3, 5455, 300),
                                                    (2, 1, 16384, 70), (1, 2, 16392, 70), (1, 1, 40001, 900), (1, 1, 70000, 2000)])
def test_against_the_formula(dtype, contexts, window, V, hist):
    check(*make(contexts, window, V, hist, dtype, seed=V))


@pytest.mark.parametrize("keep", ["bias", "allowed", "history", "none"])
def test_each_rule_alone(keep):
    x, r = make(2, 4, 300, 30, torch.float32, seed=1)
    names = {"history": ("history", "history_lens", "repetition", "presence", "frequency"), "none": ()}.get(keep, (keep,))
    check(x, {k: v for k, v in r.items() if k in names})


def test_shared_rows_and_whole_histories():
    x, r = make(4, 2, 100, 12, torch.bfloat16, seed=2)
    check(x, {**r, "bias": r["bias"][0], "allowed": r["allowed"][0], "history_lens": None})
    check(x, {"bias": r["bias"][1]})
    r["history"][:, ::2] = -1                   # no token, and tokens past the vocabulary
    r["history"][:, 1] = 100
    r["history_lens"] = torch.tensor([-3, 0, 12, 2 ** 31 - 1], dtype=torch.int32)   # clamped
    check(x, r)


def test_repeated_tokens_and_large_counts():
    x, r = make(1, 2, 50, 3000, torch.float32, seed=3)
    r["history"][:] = 7
    r["history_lens"][:] = 3000
    r["frequency"] = 1e-3
    check(x, r)
    r["history"] = torch.full((1, 65535), 6, dtype=torch.int32)      # the most that 16 bits count, beside its neighbour
    r["history"][0, :5] = 7
    r["history_lens"] = None
    check(x, r)


def test_ties_negative_penalties_and_special_values():
    import rnnt_amd

    x = torch.zeros(6, 300)
    x[0, [17, 200]] = 5.0
    x[1, 40] = math.nan                    # masked: does not count
    x[2, 41] = math.inf                    # masked
    x[3, 10] = math.nan                    # allowed: the maximum
    x[4, :] = -math.inf
    x[5, 3] = math.inf
    allowed = torch.ones(300, dtype=torch.bool)
    allowed[[40, 41]] = False
    check(x, dict(allowed=allowed))
    check(x.half(), dict(allowed=allowed, history=torch.tensor([[17, 3, 10]], dtype=torch.int32), presence=-0.5, repetition=0.5, frequency=-0.1))
    low = torch.full((2, 64), torch.finfo(torch.float32).min)
    check(low, dict(allowed=torch.arange(64) > 5))
    bias = torch.zeros(300)
    bias[17] = -math.inf                   # a banned token
    check(x[:1], dict(bias=bias))
    token, logp = rnnt_amd.row_max_logp(torch.randn(2, 70, device=DEV), rules_of(dict(allowed=torch.zeros(70, dtype=torch.bool))))
    assert token.tolist() == [0, 0] and torch.isnan(logp).all()    # a mask that leaves nothing


def test_empty_rules_are_the_plain_calls():
    import rnnt_amd

    x = torch.randn(9, 4232, device=DEV)
    token, logp = rnnt_amd.row_max_logp(x, rnnt_amd.LogitRules(history=torch.zeros(3, 0, dtype=torch.int32, device=DEV)))
    plain_token, plain_logp = rnnt_amd.row_max_logp(x)
    assert torch.equal(token, plain_token) and torch.equal(token, rnnt_amd.row_argmax(x))
    torch.testing.assert_close(logp, plain_logp, rtol=0, atol=2e-6)
    assert torch.equal(rnnt_amd.process_logits(x, rnnt_amd.LogitRules()), x)


def test_layouts():
    x, r = make(2, 2, 96, 9, torch.bfloat16, seed=4)
    import rnnt_amd

    wide = torch.cat((x, x), 1).to(DEV)[:, 96:]                  # rows apart: laid out by the call
    rules = rules_of(r)
    assert torch.equal(rnnt_amd.process_logits(wide, rules), rnnt_amd.process_logits(x.to(DEV), rules))
    flat = torch.zeros(4 * 96 + 3, dtype=torch.bfloat16, device=DEV)
    odd = flat[3:].view(4, 96)
    odd.copy_(x)
    assert torch.equal(rnnt_amd.process_logits(odd, rules), rnnt_amd.process_logits(x.to(DEV), rules))
    rules.bias = torch.cat((torch.zeros(1, device=DEV), r["bias"].to(DEV).reshape(-1)))[1:].view(2, 96)   # off 16 bytes
    assert torch.equal(rnnt_amd.process_logits(x.to(DEV), rules).cpu(), plain.rules32(x, 96, **r).to(torch.bfloat16))


def test_more_than_32_bits_of_logits():
    """33 000 rows of 70 001 bf16 logits (4.6 GB): the last rows are what the same rows alone give."""
    import rnnt_amd

    V, rows = 70001, 33000
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device=DEV)
    x[-3:] = torch.randn(3, V, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).bfloat16()
    rules = rnnt_amd.LogitRules(bias=torch.linspace(-1, 1, V, device=DEV), history=torch.full((1, 1), 5, dtype=torch.int32, device=DEV),
                                presence_penalty=3.0)
    token, logp = rnnt_amd.row_max_logp(x, rules)
    last = x[-3:].clone()
    token3, logp3 = rnnt_amd.row_max_logp(last, rules)
    assert torch.equal(token[-3:], token3) and torch.equal(logp[-3:], logp3) and int(token[0]) == V - 1
    assert rnnt_amd.process_logits(x, rules, out=x).data_ptr() == x.data_ptr()
    assert torch.equal(x[-3:], rnnt_amd.process_logits(last, rules))


def test_refusals_on_the_device():
    import rnnt_amd

    x = torch.zeros(4, 64, device=DEV)
    with pytest.raises(RuntimeError, match="bias must be on"):
        rnnt_amd.row_argmax(x, rnnt_amd.LogitRules(bias=torch.zeros(64)))
    pool = torch.zeros(4 * 64 + 8, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        rnnt_amd.process_logits(pool[:256].view(4, 64), rnnt_amd.LogitRules(), out=pool[8:].view(4, 64))
    with pytest.raises(ValueError, match="out must be"):
        rnnt_amd.process_logits(x, rnnt_amd.LogitRules(), out=torch.zeros(64, 4, device=DEV).t())
    with pytest.raises(RuntimeError, match="no backward"):
        rnnt_amd.process_logits(x.requires_grad_(True), rnnt_amd.LogitRules())


def test_captured_and_replayed():
    import rnnt_amd

    x, r = make(4, 8, 4234, 50, torch.float32, seed=6)
    xd, rules = x.to(DEV), rules_of(r)
    call = lambda: (*rnnt_amd.row_max_logp(xd, rules), rnnt_amd.process_logits(xd, rules))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in range(3):
        fresh, r2 = make(4, 8, 4234, 50, torch.float32, seed=60 + seed)
        xd.copy_(fresh)
        rules.history.copy_(r2["history"])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, call()))


def test_results_in_the_callers_buffer():
    """Nothing that the call reads may lie in it, and autograd learns that it changed."""
    import rnnt_amd

    pool = torch.zeros(4 * 64, device=DEV)
    x, out = torch.zeros(4, 64, device=DEV), pool.view(4, 64)
    words = pool.view(torch.int32)
    for rules in (rnnt_amd.LogitRules(bias=out), rnnt_amd.LogitRules(allowed=words[:2]),
                  rnnt_amd.LogitRules(history=words[-8:].view(4, 2)),
                  rnnt_amd.LogitRules(history=torch.zeros(4, 2, dtype=torch.int32, device=DEV), history_lens=words[60:64])):
        with pytest.raises(ValueError, match="must not overlap another argument"):
            rnnt_amd.process_logits(x, rules, out=out)
    leaf = torch.randn(4, 64, device=DEV, requires_grad=True)
    y = leaf * 2
    z = y.square().sum()
    with torch.no_grad():
        rnnt_amd.process_logits(y, rnnt_amd.LogitRules(presence_penalty=1.0), out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        z.backward()
    with torch.inference_mode():
        y = torch.randn(4, 64, device=DEV)
        assert rnnt_amd.process_logits(y, rnnt_amd.LogitRules(), out=y) is not None


def test_history_far_outside_the_vocabulary():
    x, r = make(2, 1, 37, 12, torch.bfloat16, seed=9)
    r["history"][:, :4] = torch.tensor([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 8, 37], dtype=torch.int32)
    r["history_lens"][:] = 12
    check(x, r)

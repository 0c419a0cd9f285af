"""GPU tests of the operators together, as they are used: PredictionNet against a 64-bit restatement, a training step of
embedding, convolution, scan, joint and transducer loss, and the greedy searches over a PredictionNet under rules."""
import pytest
import torch
import torch.nn.functional as F

import plain_operators as plain

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def plain_net(p, tokens, lens, width, state, scale=1.0):
    """PredictionNet.forward in 64 bits on the CPU from its state dict (differentiable: torch operations only)."""
    u = p["embedding.weight"][tokens] * scale
    for i in range(sum(k.endswith("A_log") for k in p)):
        q = {k.split(".", 2)[2]: v for k, v in p.items() if k.startswith(f"layers.{i}.")}
        inner = q["D"].shape[0]
        x, z = (F.layer_norm(u, u.shape[-1:], q["norm.weight"], q["norm.bias"]) @ q["in_proj.weight"].t()).split(inner, -1)
        pad = F.pad(x, (0, 0, width - 1, 0))
        c = sum(pad[:, k:k + x.shape[1]] * q["conv_weight"][:, k] for k in range(width)) + q["conv_bias"]
        c = c * torch.sigmoid(c)
        live = (torch.arange(x.shape[1])[None] < lens[:, None]).double()[..., None]
        c = c * live
        rank = q["dt_proj.weight"].shape[1]
        r, B, C = (c @ q["x_proj.weight"].t()).split((rank, state, state), -1)
        delta = F.softplus(r @ q["dt_proj.weight"].t() + q["dt_bias"])
        A = -torch.exp(q["A_log"])
        h, ys = torch.zeros(x.shape[0], inner, state, dtype=u.dtype), []
        for t in range(x.shape[1]):
            h = torch.exp(delta[:, t, :, None] * A) * h + (delta[:, t] * c[:, t])[..., None] * B[:, t, None]
            ys.append((h * C[:, t, None]).sum(-1) + q["D"] * c[:, t])
        y = torch.stack(ys, 1) * z * torch.sigmoid(z) * live
        u = u + y @ q["out_proj.weight"].t()
    return F.layer_norm(u, u.shape[-1:], p["norm.weight"], p["norm.bias"]) @ p["output_proj.weight"].t() + p["output_proj.bias"]


def make_net(V=29, E=24, out=16, layers=2, seed=0, **kw):
    import rnnt_amd

    torch.manual_seed(seed)
    return rnnt_amd.PredictionNet(V, E, out, layers=layers, **kw)


@pytest.mark.parametrize("state,width,layers", [(16, 4, 2), (8, 2, 1), (32, 3, 1)])
def test_forward_and_gradients_against_64_bits(state, width, layers):
    net = make_net(state_size=state, conv_width=width, layers=layers, embed_scale="sqrt")
    tokens = torch.randint(0, 29, (3, 11), generator=torch.Generator().manual_seed(1))
    tokens[:, 0] = 0
    lens = torch.tensor([11, 4, 1])
    go = torch.randn(3, 11, 16, generator=torch.Generator().manual_seed(2))
    live = (torch.arange(11)[None] < lens[:, None])
    go[~live] = 0
    p = {k: v.detach().double().requires_grad_(True) for k, v in net.state_dict().items()}
    ref = plain_net(p, tokens, lens, width, state, 24 ** 0.5)
    ref.backward(go.double())
    net = net.to(DEV)
    out, _ = net(tokens.to(DEV), length=lens.to(DEV))
    out.backward(go.to(DEV))
    # some twenty fp32 products and norms in a row, each within a few dozen u of values of order one
    torch.testing.assert_close(out.detach().cpu().double()[live], ref.detach()[live], rtol=2e-5, atol=2e-5)
    for k, v in net.named_parameters():
        want = p[k].grad if k != "embedding.weight" else p[k].grad.index_fill(0, torch.tensor([0]), 0.0)
        err = float((v.grad.cpu().double() - want).norm() / want.norm().clamp(min=1e-12))
        assert err < 2e-5, (k, err)


@pytest.mark.parametrize("amp", [torch.bfloat16, torch.float16])
def test_under_autocast(amp):
    """fp32 parameters, 16-bit sequences: gradients in fp32, near the fp32 step's."""
    net = make_net().to(DEV)
    tokens = torch.randint(0, 29, (3, 9), generator=torch.Generator().manual_seed(1)).to(DEV)
    go = torch.randn(3, 9, 16, generator=torch.Generator().manual_seed(2)).to(DEV)
    grads = []
    for on in (False, True):
        net.zero_grad()
        with torch.autocast("cuda", dtype=amp, enabled=on):
            out, _ = net(tokens)
        assert out.dtype is (amp if on else torch.float32)
        out.float().backward(go)
        grads.append([p.grad.clone() for p in net.parameters()])
    for (name, _), a, b in zip(net.named_parameters(), *grads):
        assert b.dtype is torch.float32
        # a dozen tensors on the way are rounded by half a step of the type each
        assert float((a - b).norm()) <= 16 * torch.finfo(amp).eps * float(a.norm()) + 1e-6, name


def test_hidden_carries_a_sequence_on():
    net = make_net().to(DEV).eval()
    tokens = torch.randint(0, 29, (2, 9), device=DEV)
    with torch.no_grad():
        whole, hidden = net(tokens)
        part, h = net(tokens[:, :4])
        outs = [part]
        for t in range(4, 9):
            kept = tuple(x.clone() for x in h)
            o, nxt = net(tokens[:, t:t + 1], hidden=h)
            assert all(torch.equal(a, b) for a, b in zip(h, kept))          # the caller's hidden is not changed
            h = nxt
            outs.append(o)
    torch.testing.assert_close(torch.cat(outs, 1), whole, rtol=2e-5, atol=2e-5)
    for a, b in zip(h, hidden):
        torch.testing.assert_close(a, b, rtol=2e-5, atol=2e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_step_to_the_transducer_loss(dtype):
    """labels -> PredictionNet -> JointNet.transducer_loss -> gradients, against the same step in 64 bits on the CPU with the
    loss from log-probabilities by dynamic programming."""
    import rnnt_amd

    B, T, U, V, He, Hd = 2, 7, 4, 29, 12, 16
    net = make_net(V=V, E=24, out=Hd, layers=1)
    joint = rnnt_amd.JointNet(He + Hd, 20, V)
    g = torch.Generator().manual_seed(5)
    enc = torch.randn(B, T, He, generator=g)
    labels = torch.randint(1, V, (B, U), generator=g, dtype=torch.int32)
    act_lens, label_lens = torch.tensor([7, 5], dtype=torch.int32), torch.tensor([4, 2], dtype=torch.int32)
    if dtype is torch.bfloat16:       # the same rounded inputs and parameters on both sides
        net, joint, enc = net.to(dtype), joint.to(dtype), enc.to(dtype)
    p = {k: v.detach().double().requires_grad_(True) for k, v in net.state_dict().items()}
    j = {k: v.detach().double() for k, v in joint.state_dict().items()}
    inputs = F.pad(labels, (1, 0)).long()
    dec = plain_net(p, inputs, label_lens.long() + 1, 4, 16)
    hid = torch.tanh(torch.cat((enc.double()[:, :, None].expand(B, T, U + 1, He), dec[:, None].expand(B, T, U + 1, Hd)), -1) @ j["mlp.0.weight"].t()
                     + j["mlp.0.bias"])
    lp = F.log_softmax(hid @ j["mlp.2.weight"].t() + j["mlp.2.bias"], -1)
    loss = 0
    for b in range(B):
        alpha = {(0, 0): lp.new_zeros(())}
        for t in range(int(act_lens[b])):
            for u in range(int(label_lens[b]) + 1):
                come = []
                if t:
                    come.append(alpha[t - 1, u] + lp[b, t - 1, u, 0])
                if u:
                    come.append(alpha[t, u - 1] + lp[b, t, u - 1, labels[b, u - 1]])
                if come:
                    alpha[t, u] = torch.logsumexp(torch.stack(come), 0)
        loss = loss - (alpha[int(act_lens[b]) - 1, int(label_lens[b])] + lp[b, int(act_lens[b]) - 1, int(label_lens[b]), 0])
    (loss / B).backward()
    net, joint = net.to(DEV), joint.to(DEV)
    out, _ = net(inputs.to(DEV), length=(label_lens + 1).to(DEV))
    got = joint.transducer_loss(enc.to(DEV), out, labels.to(DEV), act_lens, label_lens)
    got.sum().backward()
    # fp32: dozens of roundings of 2^-24; bf16: every tensor between the operators is rounded (2^-9 each, a dozen in a row)
    tol = 1e-4 if dtype is torch.float32 else 6e-2
    assert float(got.detach()) == pytest.approx(float(loss.detach()) / B, rel=tol)
    for k, v in net.named_parameters():
        want = p[k].grad if k != "embedding.weight" else p[k].grad.index_fill(0, torch.tensor([0]), 0.0)
        err = float((v.grad.cpu().double() - want).norm() / want.norm().clamp(min=1e-9))
        assert err < (1e-4 if dtype is torch.float32 else 0.15), (k, err)


def _joint(He, Hd, V, seed):
    import rnnt_amd

    torch.manual_seed(seed)
    joint = rnnt_amd.JointNet(He + Hd, 32, V).to(DEV)
    with torch.no_grad():
        joint.mlp[2].bias[0] += 1.0
        joint.mlp[2].weight *= 3.0
    return joint


def _search_frame_by_frame(enc, net, joint, rules, V):
    """One utterance, one frame at a time, the rules by the formula."""
    tokens = []
    dec, hidden = net(torch.zeros(1, 1, dtype=torch.long, device=DEV))
    for t in range(enc.shape[0]):
        row = joint(enc[t], dec[0, 0])[None].float()
        hist = torch.tensor([tokens], dtype=torch.int32) if tokens else None
        allowed = rules["allowed"](tokens) if callable(rules.get("allowed")) else rules.get("allowed")
        want = plain.rules32(row, V, bias=rules.get("bias"), allowed=allowed, history=hist, repetition=rules.get("repetition", 1.0),
                             presence=rules.get("presence", 0.0), frequency=rules.get("frequency", 0.0))
        best = int(want.argmax())
        if best:
            tokens.append(best)
            dec, hidden = net(torch.tensor([[best]], device=DEV), hidden=hidden)
    return tokens


@pytest.mark.parametrize("kind", ["none", "penalties", "bias", "grammar", "all"])
def test_greedy_searches_under_rules(kind):
    import rnnt_amd

    V, He, Hd, T, B = 31, 12, 16, 40, 3
    net, joint = make_net(V=V, out=Hd, layers=1, seed=3).to(DEV).eval(), _joint(He, Hd, V, 4)
    enc = torch.randn(B, T, He, device=DEV, generator=torch.Generator(device=DEV).manual_seed(9)) * 2
    no_repeat = lambda tokens: torch.tensor([v == 0 or not tokens or v != tokens[-1] for v in range(V)])  # noqa: E731
    r = {}
    if kind in ("penalties", "all"):
        r.update(repetition=1.4, presence=0.3, frequency=0.2)
    if kind in ("bias", "all"):
        r["bias"] = torch.zeros(V).index_fill(0, torch.tensor([5, 6]), 2.0).index_fill(0, torch.tensor([7]), -float("inf"))
    if kind in ("grammar", "all"):
        r["allowed"] = no_repeat
    rules = rnnt_amd.LogitRules(bias=r["bias"].to(DEV) if "bias" in r else None,
                                allowed=(lambda tokens: rnnt_amd.pack_allowed(no_repeat(tokens))) if "allowed" in r else None,
                                repetition_penalty=r.get("repetition", 1.0), presence_penalty=r.get("presence", 0.0),
                                frequency_penalty=r.get("frequency", 0.0))
    with torch.no_grad():
        want = [_search_frame_by_frame(enc[b], net, joint, r, V) for b in range(B)]
        batch, _, _, _ = rnnt_amd.greedy_search_batch(enc, net, joint, window=7, rules=rules)
        single = [rnnt_amd.greedy_decode(enc[b], T, net, joint, window=5, rules=rules) for b in range(B)]
    assert any(want)
    assert batch == want and single == want
    if kind in ("bias", "all"):
        assert all(7 not in w for w in want)
    if kind in ("grammar", "all"):
        assert all(a != b for w in want for a, b in zip(w, w[1:]))


def test_a_given_history_counts_and_a_callable_mask_is_for_searches():
    import rnnt_amd

    V, He, Hd = 31, 12, 16
    net, joint = make_net(V=V, out=Hd, layers=1, seed=3).to(DEV).eval(), _joint(He, Hd, V, 4)
    enc = torch.randn(2, 20, He, device=DEV, generator=torch.Generator(device=DEV).manual_seed(9)) * 2
    free, _, _, _ = rnnt_amd.greedy_search_batch(enc, net, joint)
    said = sorted(set(sum(free, [])))
    assert said
    history = torch.tensor([said, said], dtype=torch.int32, device=DEV)
    rules = rnnt_amd.LogitRules(history=history, presence_penalty=1e4)
    got, _, _, _ = rnnt_amd.greedy_search_batch(enc, net, joint, rules=rules)
    assert not set(sum(got, [])) & set(said)
    rules = rnnt_amd.LogitRules(history=history, history_lens=torch.zeros(2, dtype=torch.int32, device=DEV), presence_penalty=1e4)
    got, _, _, _ = rnnt_amd.greedy_search_batch(enc, net, joint, rules=rules)
    assert got[0][:1] == free[0][:1]                     # nothing counted yet at the first emission
    with pytest.raises(ValueError, match="rules.bias"):
        rnnt_amd.greedy_search_batch(enc, net, joint, rules=rnnt_amd.LogitRules(bias=torch.zeros(3, device=DEV)))
    with pytest.raises(ValueError, match="rules.history"):
        rnnt_amd.greedy_search_batch(enc, net, joint, rules=rnnt_amd.LogitRules(history=history[:1]))


def test_capture_is_refused_while_an_eager_graph_holds_the_parameters():
    """Refused before anything is launched; once the eager results are gone the same pass is captured and replayed."""
    import rnnt_amd

    tokens = torch.randint(0, 12, (3, 5), device=DEV)
    weight = torch.randn(12, 64, device=DEV, requires_grad=True)
    taps = torch.randn(64, 4, device=DEV, requires_grad=True)
    dt, A, B = torch.randn(3, 5, 64, device=DEV), -torch.rand(64, 8, device=DEV), torch.randn(3, 5, 8, device=DEV)
    A.requires_grad_(True)

    def run():
        x = rnnt_amd.token_embedding(tokens, weight)
        y, _ = rnnt_amd.causal_conv(x, taps)
        z, _ = rnnt_amd.selective_scan(y, dt, A, B, B)
        return (z, *torch.autograd.grad(z, (weight, taps, A), torch.ones_like(z)))

    fixed = torch.randn(3, 5, 64, device=DEV)
    calls = (lambda: rnnt_amd.token_embedding(tokens, weight), lambda: rnnt_amd.causal_conv(fixed, taps)[0],
             lambda: rnnt_amd.selective_scan(fixed, dt, A, B, B)[0])
    for call in calls:
        held = call()
        graph, scratch = torch.cuda.CUDAGraph(), torch.zeros(1, device=DEV)
        with torch.cuda.graph(graph):
            scratch.add_(1)
            with pytest.raises(RuntimeError, match="cannot be captured while"):
                call()
        del held
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(3):
        tokens.copy_(torch.randint(0, 12, (3, 5), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            eager = run()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager))

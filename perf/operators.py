"""What is measured of the prediction network's and the decoder's operators: token embedding, causal convolution,
selective scan (training, prompts, single tokens) and decoding rules on logits, each in its plain form (``own``
false) and through this package's calls (``own`` true)."""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the label sequences of one training batch (32 utterances of 40 labels and the start symbol) into the
        # prediction network, forward and backward
        dict(name="embed_labels", op="embed", rows=32, length=41, vocab=4232, dim=512, type="bf16", padding=True),
        # text-only training of the prediction network: many lines at once, frequent words, a sixth of it padding
        dict(name="embed_text", op="embed", rows=128, length=511, vocab=16384, dim=512, type="f32", padding=True),
        # the same label sequences through the short convolution; its single-token form for one utterance; frames of
        # long utterances (T = 1500) through an encoder layer
        dict(name="conv_step_one", op="conv_step", rows=1, dim=1024, width=4, type="bf16"),
        dict(name="conv_train_frames", op="conv_train", rows=16, length=1500, dim=1024, width=4, type="f16"),
        # the scan in training: label sequences, and the frames of long utterances
        dict(name="scan_train_labels", op="scan_train", rows=32, length=41, dim=1024, state=16, type="bf16"),
        dict(name="scan_train_frames", op="scan_train", rows=16, length=1500, dim=1024, state=16, type="bf16"),
        # a long text prompt of one user, continued from a cached state
        dict(name="scan_prompt_long", op="scan_prompt", rows=1, length=4095, dim=1536, state=16, type="f32"),
        # one emission of one utterance, and of a large decoding batch
        dict(name="scan_step_one", op="scan_step", rows=1, dim=1024, state=16, type="bf16"),
        dict(name="scan_step_batch", op="scan_step", rows=256, dim=2048, state=16, type="bf16"),
        # one utterance's single frame under a hotword bias and penalties; a window of 32 frames for 16 utterances with
        # all rules; the processed logits of a large vocabulary for a caller that samples
        dict(name="pick_one", op="pick", contexts=1, window=1, vocab=5455, history=37, type="f16"),
        dict(name="pick_window", op="pick", contexts=16, window=32, vocab=4232, history=151, type="f32"),
        dict(name="process_large", op="process", contexts=64, window=1, vocab=70001, history=1500, type="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "conv_step", "conv_train", "scan_train", "scan_prompt", "scan_step", "pick", "process"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op == "embed":
        length = _log(rng, 1, 1500)
        rows = _log(rng, 1, max(1, min(128, 65408 // length)))
        return dict(op=op, rows=rows, length=length, vocab=_log(rng, 30, 16384), dim=_log(rng, 64, 512), type=kind,
                    padding=rng.random() < 0.5)
    if op == "conv_step":
        return dict(op=op, rows=_log(rng, 1, 256), dim=_log(rng, 64, 2048), width=rng.choice([2, 3, 4]), type=kind)
    if op == "conv_train":
        dim = _log(rng, 64, 2048)
        length = _log(rng, 1, 2048)
        rows = _log(rng, 1, max(1, min(64, 16 * 1500 * 512 // (dim * length))))
        return dict(op=op, rows=rows, length=length, dim=dim, width=rng.choice([2, 3, 4]), type=kind)
    if op in ("scan_train", "scan_prompt"):
        state = rng.choice([8, 16, 32])
        dim = _log(rng, 64, 2048)
        length = _log(rng, 1, 4096)
        rows = _log(rng, 1, max(1, min(64, 16 * 1500 * 1024 * 8 // (dim * length * state))))
        return dict(op=op, rows=rows, length=length, dim=dim, state=state, type=kind)
    if op == "scan_step":
        return dict(op=op, rows=_log(rng, 1, 256), dim=_log(rng, 64, 2048), state=rng.choice([8, 16, 32]), type=kind)
    vocab = _log(rng, 30, 70001)
    contexts = _log(rng, 1, max(1, min(64, 4480064 // vocab)))
    window = _log(rng, 1, max(1, min(64, 4480064 // (vocab * contexts)))) if op == "pick" else 1
    return dict(op=op, contexts=contexts, window=window, vocab=vocab, history=_log(rng, 1, 1500), type=kind)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    kind = _TYPES[case["type"]]
    op = case["op"]

    def randn(*shape, scale=1.0, dtype=kind):
        return (torch.randn(*shape, device=dev, generator=g) * scale).to(dtype)

    def rand(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, device=dev, generator=g) * (hi - lo) + lo

    def lengths(rows, length):
        # one sequence fills the tensor, the others are between a quarter of it and all of it
        n = (rand(rows, lo=0.25, hi=1.0) * length).ceil().clamp(1, length).to(torch.int32)
        n[0] = length
        return n

    s = {"case": case}
    if op == "embed":
        n, v = (case["rows"], case["length"]), case["vocab"]
        s["tokens"] = (rand(*n).pow(3) * v).long().clamp(0, v - 1)   # frequent and rare tokens
        if case["padding"]:
            s["tokens"].masked_fill_(torch.arange(n[1], device=dev) >= lengths(*n)[:, None], 0)
        s["padding"] = 0 if case["padding"] else None
        s["scale"] = math.sqrt(case["dim"])
        s["weight"] = randn(v, case["dim"], scale=1.0 / math.sqrt(case["dim"]))
        s["grad"] = randn(*n, case["dim"])
        return s
    if op in ("conv_step", "conv_train"):
        rows, dim, width = case["rows"], case["dim"], case["width"]
        s["weight"] = randn(dim, width, scale=1.0 / math.sqrt(width), dtype=torch.float32)
        s["bias"] = randn(dim, scale=0.1, dtype=torch.float32)
        if op == "conv_step":
            s["x"], s["state"] = randn(rows, dim), randn(rows, width - 1, dim)
        else:
            # one half of what the layer's input projection gives, as a view
            s["x"] = randn(rows, case["length"], 2 * dim)[..., :dim]
            s["grad"] = randn(rows, case["length"], dim)
            s["lengths"] = lengths(rows, case["length"])
        return s
    if op.startswith("scan"):
        rows, dim, state = case["rows"], case["dim"], case["state"]
        lead = (rows,) if op == "scan_step" else (rows, case["length"])
        s["x"] = randn(*lead, dim)
        s["dt"] = randn(*lead, dim, scale=0.5)
        s["z"] = randn(*lead, 2 * dim)[..., dim:]                    # the other half of the input projection
        rank = max(1, dim // 16)
        wide = randn(*lead, rank + 2 * state)                        # B and C are parts of one projection's output
        s["B"], s["C"] = wide[..., rank:rank + state], wide[..., rank + state:]
        s["A"] = -(torch.arange(1, state + 1, device=dev).float() * rand(dim, 1, lo=0.7, hi=1.3))
        s["D"] = 1.0 + 0.1 * randn(dim, dtype=torch.float32)
        s["bias"] = torch.log(torch.expm1(rand(dim, lo=math.log(1e-3), hi=math.log(1e-1)).exp()))
        if op == "scan_train":
            s["grad"] = randn(*lead, dim)
        else:
            s["state"] = randn(rows, dim, state, dtype=torch.float32)
        if op != "scan_step":
            s["lengths"] = lengths(rows, case["length"])
        return s
    contexts, v, words = case["contexts"], case["vocab"], (case["vocab"] + 31) // 32
    s["x"] = randn(contexts * case["window"], v, scale=3.0)
    s["history"] = (rand(contexts, case["history"]).pow(2) * v).int().clamp(0, v - 1)
    s["history_lens"] = lengths(contexts, case["history"])
    s["bias"] = randn(contexts, v, dtype=torch.float32) * (rand(contexts, v) < 0.05)          # boosted and banned words
    bits = (rand(contexts, words * 32) < 0.9).view(contexts, words, 32)
    word = (bits.long() << torch.arange(32, device=dev)).sum(-1)
    s["allowed"] = torch.where(word >= 2 ** 31, word - 2 ** 32, word).int()                   # one bit for a token
    s["repetition"], s["presence"], s["frequency"] = 1.25, 0.3, 0.15
    s["divisor"] = torch.tensor(s["repetition"], device=dev)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return _own(op, s)
    if op == "embed":
        return _embed(s)
    if op == "conv_step":
        return _conv_step(s)
    if op == "conv_train":
        return _conv_train(s)
    if op == "scan_step":
        return _scan_step(s)
    if op.startswith("scan"):
        return _scan(s, op == "scan_train")
    return _rules(s, op == "pick")


def _own(op, s):
    import rnnt_amd

    if op == "embed":
        w = s["weight"].detach().requires_grad_(True)
        out = rnnt_amd.token_embedding(s["tokens"], w, scale=s["scale"], padding_idx=s["padding"])
        return {"out": out.detach(), "dweight": torch.autograd.grad(out, w, s["grad"])[0]}
    if op == "conv_step":
        y, state = rnnt_amd.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"])
        return {"y": y, "state": state}
    if op == "conv_train":
        leaves = [s[k].detach().requires_grad_(True) for k in ("x", "weight", "bias")]
        y, _ = rnnt_amd.causal_conv(*leaves, lengths=s["lengths"])
        return dict(zip(("y", "dx", "dweight", "dbias"), (y.detach(), *torch.autograd.grad(y, leaves, s["grad"]))))
    if op == "scan_step":
        y, state = rnnt_amd.selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"],
                                                dt_bias=s["bias"])
        return {"y": y, "state": state}
    if op == "scan_prompt":
        with torch.no_grad():
            y, state = rnnt_amd.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["bias"],
                                               initial_state=s["state"], lengths=s["lengths"])
        return {"y": y, "state": state}
    if op == "scan_train":
        names = ("x", "dt", "A", "B", "C", "D", "z", "bias")
        leaves = [s[k].detach().requires_grad_(True) for k in names]
        x, dt, A, B, C, D, z, bias = leaves
        y, _ = rnnt_amd.selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=bias, lengths=s["lengths"])
        grads = torch.autograd.grad(y, leaves, s["grad"])
        return {"y": y.detach(), **{"d" + k: v for k, v in zip(names, grads)}}
    rules = rnnt_amd.LogitRules(bias=s["bias"], allowed=s["allowed"], history=s["history"], history_lens=s["history_lens"],
                                repetition_penalty=s["repetition"], presence_penalty=s["presence"],
                                frequency_penalty=s["frequency"])
    if op == "pick":
        token, logp = rnnt_amd.row_max_logp(s["x"], rules)
        return {"token": token, "logp": logp}
    return rnnt_amd.process_logits(s["x"], rules)


# the plain forms ------------------------------------------------------------------------------------------------------
def _embed(s):
    tokens, weight = s["tokens"], s["weight"]
    out = (weight.float()[tokens] * s["scale"]).to(weight.dtype)
    flat = tokens.reshape(-1)
    dweight = torch.zeros(weight.shape, device=weight.device)
    dweight.index_add_(0, flat, s["grad"].reshape(-1, weight.shape[1]).float() * s["scale"])
    if s["padding"] is not None:
        dweight[s["padding"]] = 0.0
    return {"out": out, "dweight": dweight.to(weight.dtype)}


def _taps(xe, length, width):
    return torch.stack([xe[:, k:k + length] for k in range(width)], dim=-1)       # [rows, length, dim, width]


def _conv_step(s):
    xe = torch.cat((s["state"].float(), s["x"].float()[:, None]), dim=1)
    p = (xe * s["weight"].t()).sum(1) + s["bias"]
    return {"y": (p * torch.sigmoid(p)).to(s["x"].dtype), "state": xe[:, 1:].to(s["x"].dtype)}


def _valid(s, length):
    return (torch.arange(length, device=s["lengths"].device) < s["lengths"][:, None])[..., None]


def _conv_train(s):
    x, w = s["x"], s["weight"]
    rows, length, dim = x.shape
    width = w.shape[1]
    valid = _valid(s, length)
    xe = torch.cat((torch.zeros(rows, width - 1, dim, device=x.device), torch.where(valid, x.float(), 0.0)), dim=1)
    taps = _taps(xe, length, width)
    p = (taps * w).sum(-1) + s["bias"]
    sig = torch.sigmoid(p)
    y = torch.where(valid, p * sig, 0.0)
    gp = torch.where(valid, s["grad"].float() * (sig + p * sig * (1.0 - sig)), 0.0)
    late = torch.cat((gp, torch.zeros(rows, width - 1, dim, device=x.device)), dim=1)
    dx = torch.where(valid, (_taps(late, length, width) * w.flip(1)).sum(-1), 0.0)
    return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dweight": (gp[..., None] * taps).sum((0, 1)), "dbias": gp.sum((0, 1))}


def _softplus(v):
    return torch.where(v > 20.0, v, torch.log1p(torch.exp(v.clamp(max=20.0))))


def _scan_step(s):
    x, z = s["x"].float(), s["z"].float()
    delta = _softplus(s["dt"].float() + s["bias"])
    h = torch.exp(delta[..., None] * s["A"]) * s["state"] + (delta * x)[..., None] * s["B"].float()[:, None]
    y = (h * s["C"].float()[:, None]).sum(-1) + s["D"] * x
    return {"y": (y * z * torch.sigmoid(z)).to(s["x"].dtype), "state": h}


def _recur(a, u):
    """h_t = a_t h_{t-1} + u_t along dim 1, from zero, by doubling the distance that each position has summed over."""
    k = 1
    while k < a.shape[1]:
        u = torch.cat((u[:, :k], u[:, k:] + a[:, k:] * u[:, :-k]), dim=1)
        a = torch.cat((a[:, :k], a[:, k:] * a[:, :-k]), dim=1)
        k *= 2
    return u


def _scan(s, train):
    kind, length = s["x"].dtype, s["x"].shape[1]
    valid = _valid(s, length)
    x, z = torch.where(valid, s["x"].float(), 0.0), s["z"].float()
    pre = s["dt"].float() + s["bias"]
    delta = torch.where(valid, _softplus(pre), 0.0)       # a step of length zero leaves the state as it is
    A, B, C, D = s["A"], s["B"].float(), s["C"].float(), s["D"]
    a = torch.exp(delta[..., None] * A)
    u = (delta * x)[..., None] * B[:, :, None]
    if not train:
        u[:, 0] += a[:, 0] * s["state"]
    h = _recur(a, u)
    del u
    y = (h * C[:, :, None]).sum(-1) + D * x
    sig = torch.sigmoid(z)
    out = torch.where(valid, y * z * sig, 0.0).to(kind)
    if not train:
        return {"y": out, "state": h[:, -1].contiguous()}
    grad = torch.where(valid, s["grad"].float(), 0.0)
    gy = grad * z * sig
    dC = (h * gy[..., None]).sum(2)
    ahead = torch.cat((a[:, 1:], torch.ones_like(a[:, :1])), dim=1)
    G = _recur(ahead.flip(1), (C[:, :, None] * gy[..., None]).flip(1)).flip(1)
    del ahead
    dB = (G * (delta * x)[..., None]).sum(2)
    inner = (G * B[:, :, None]).sum(-1)
    before = torch.cat((torch.zeros_like(h[:, :1]), h[:, :-1]), dim=1)
    del h
    G = G * before * a
    del before, a
    dA = (G * delta[..., None]).sum((0, 1))
    ddelta = (G * A).sum(-1) + inner * x
    ddt = torch.where(valid, ddelta * torch.sigmoid(pre), 0.0)
    dz = grad * y * (sig + z * sig * (1.0 - sig))
    return {"y": out, "dx": (inner * delta + gy * D).to(kind), "ddt": ddt.to(kind), "dA": dA, "dB": dB.to(kind), "dC": dC.to(kind),
            "dD": (gy * x).sum((0, 1)), "dz": dz.to(kind), "dbias": ddt.sum((0, 1))}


def _counts(s, dtype):
    contexts, width = s["history"].shape
    live = torch.arange(width, device=s["history"].device) < s["history_lens"][:, None]
    zero = torch.zeros(contexts, s["x"].shape[1], device=s["x"].device, dtype=dtype)
    return zero.scatter_add_(1, s["history"].long(), live.to(dtype))


def _bits(s):
    shifts = torch.arange(32, device=s["allowed"].device, dtype=torch.int32)
    bits = (s["allowed"][..., None] >> shifts) & 1
    return bits.reshape(bits.shape[0], -1)[:, :s["x"].shape[1]].bool()


def _rules(s, pick):
    window = s["case"]["window"]
    count, bias, allowed = (v.repeat_interleave(window, 0) for v in (_counts(s, torch.float32), s["bias"], _bits(s)))
    v = s["x"].float()
    v = torch.where(count > 0, torch.where(v > 0, v / s["divisor"], v * s["repetition"]), v)
    v = v - s["frequency"] * count - s["presence"] * (count > 0).float() + bias
    v = torch.where(allowed, v, -math.inf)
    if not pick:
        return v.to(s["x"].dtype)
    top = v.max(1, keepdim=True).values
    order = torch.arange(v.shape[1], device=v.device, dtype=torch.int32)
    token = torch.where(v == top, order, v.shape[1]).min(1).values
    return {"token": token, "logp": -torch.log(torch.exp(v - top).sum(1))}


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["type"] == "f32" else 2
    op = case["op"]
    if op == "embed":
        n, v, d = case["rows"] * case["length"], case["vocab"], case["dim"]
        return {"bytes": 2 * 8 * n + (min(n, v) * d + n * d) * e + (n * d + v * d) * e, "flops": 3 * n * d}
    if op == "conv_step":
        n, w = case["rows"] * case["dim"], case["width"]
        return {"bytes": n * 2 * w * e + case["dim"] * (w + 1) * 4, "flops": n * (2 * w + 5)}
    if op == "conv_train":
        n, w = case["rows"] * case["length"] * case["dim"], case["width"]
        return {"bytes": 5 * n * e + case["dim"] * (w + 1) * 12, "flops": n * (8 * w + 16)}
    if op == "scan_step":
        r, d, n = case["rows"], case["dim"], case["state"]
        return {"bytes": r * (4 * d * e + 2 * n * e + 8 * d * n) + 4 * d * (n + 2), "flops": 7 * r * d * n}
    if op.startswith("scan"):
        r, d, n, t = case["rows"], case["dim"], case["state"], case["length"]
        ends = 4 * d * (n + 2)
        if op == "scan_prompt":
            return {"bytes": r * t * (4 * d + 2 * n) * e + 8 * r * d * n + ends, "flops": 7 * r * t * d * n}
        return {"bytes": r * t * (11 * d + 6 * n) * e + 3 * ends, "flops": 24 * r * t * d * n}
    c, v, r = case["contexts"], case["vocab"], case["contexts"] * case["window"]
    given = c * (4 * v + (v + 31) // 32 * 4 + 4 * case["history"])
    return {"bytes": r * v * e + given + (8 * r if op == "pick" else r * v * e), "flops": 8 * r * v}


# ---------------------------------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if op == "embed":
        flat, g = s["tokens"].reshape(-1), f["grad"].reshape(-1, case["dim"])
        dweight = torch.zeros(case["vocab"], case["dim"], device=g.device, dtype=torch.float64)
        keep = torch.ones_like(flat, dtype=torch.bool) if s["padding"] is None else flat != s["padding"]
        dweight.index_put_((flat[keep],), g[keep], accumulate=True)
        return {"out": torch.index_select(f["weight"], 0, flat).reshape(f["grad"].shape) * s["scale"], "dweight": dweight * s["scale"]}
    if op == "conv_step":
        w = case["width"]
        p = f["bias"] + f["x"] * f["weight"][:, w - 1]
        for k in range(w - 1):
            p = p + f["state"][:, k] * f["weight"][:, k]
        return {"y": p / (1 + torch.exp(-p)), "state": torch.cat((f["state"], f["x"][:, None]), 1)[:, 1:]}
    if op == "conv_train":
        return _exact_conv(s, f, case["width"])
    if op == "scan_step":
        wide = {k: f[k][:, None] for k in ("x", "dt", "z", "B", "C")}
        y, _, state, _ = _exact_states(wide, f, f["state"], torch.ones(case["rows"], device=f["x"].device, dtype=torch.int32), keep=False)
        return {"y": y[:, 0] * f["z"] / (1 + torch.exp(-f["z"])), "state": state}
    if op == "scan_prompt":
        y, _, state, live = _exact_states(f, f, f["state"], s["lengths"], keep=False)
        return {"y": y * f["z"] / (1 + torch.exp(-f["z"])) * live, "state": state}
    if op == "scan_train":
        return _exact_train(s, f)
    count = torch.zeros(case["contexts"], case["vocab"], device=f["x"].device, dtype=torch.float64)
    live = (torch.arange(case["history"], device=f["x"].device) < s["history_lens"][:, None]).double()
    count.scatter_add_(1, s["history"].long(), live)
    word, bit = torch.arange(case["vocab"], device=f["x"].device) // 32, torch.arange(case["vocab"], device=f["x"].device) % 32
    allowed = (s["allowed"].long()[:, word] >> bit) & 1
    v = f["x"].view(case["contexts"], case["window"], case["vocab"])
    count, bias, allowed = count[:, None], f["bias"][:, None], allowed[:, None]
    seen = torch.where(v > 0, v / s["repetition"], v * s["repetition"]) - s["presence"]
    v = torch.where(count > 0, seen, v) - s["frequency"] * count + bias
    v = v.masked_fill(allowed == 0, -math.inf).view(-1, case["vocab"])
    if op == "pick":
        return {"token": None, "logp": v.amax(1) - torch.logsumexp(v, 1)}
    return v


def _exact_conv(s, f, width):
    x, w, g = f["x"], f["weight"], f["grad"]
    rows, length, dim = x.shape
    y, dx = torch.zeros_like(g), torch.zeros(rows, length, dim, device=x.device, dtype=torch.float64)
    dw, db = torch.zeros_like(w), torch.zeros_like(f["bias"])
    for b in range(rows):
        n = int(s["lengths"][b])
        p = f["bias"].expand(n, dim).clone()
        for back in range(min(width, n)):
            p[back:] += x[b, :n - back] * w[:, width - 1 - back]
        sig = 1 / (1 + torch.exp(-p))
        y[b, :n] = p * sig
        gp = g[b, :n] * sig * (1 + p * (1 - sig))
        db += gp.sum(0)
        for back in range(min(width, n)):
            dx[b, :n - back] += gp[back:] * w[:, width - 1 - back]
            dw[:, width - 1 - back] += (gp[back:] * x[b, :n - back]).sum(0)
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


def _exact_states(seq, f, state, lens, keep):
    """y before the gate, every state where ``keep``, the last state and which positions are live."""
    rows, length, dim = seq["x"].shape
    live = (torch.arange(length, device=lens.device) < lens[:, None]).double()[..., None]
    delta = torch.logaddexp(seq["dt"] + f["bias"], torch.zeros((), device=lens.device, dtype=torch.float64)) * live
    y, states, h = torch.zeros_like(seq["x"]), [], state
    for t in range(length):
        h = h * torch.exp(delta[:, t, :, None] * f["A"]) + (delta[:, t] * seq["x"][:, t])[..., None] * seq["B"][:, t, None, :]
        y[:, t] = (h @ seq["C"][:, t, :, None])[..., 0] + f["D"] * seq["x"][:, t]
        if keep:
            states.append(h)
    return y, states, h, live


def _exact_train(s, f):
    rows, length, dim = f["x"].shape
    n = f["A"].shape[1]
    start = torch.zeros(rows, dim, n, device=f["x"].device, dtype=torch.float64)
    y, states, _, live = _exact_states(f, f, start, s["lengths"], keep=True)
    gate = 1 / (1 + torch.exp(-f["z"]))
    g = f["grad"] * live
    gy = g * f["z"] * gate
    pre = f["dt"] + f["bias"]
    delta = torch.logaddexp(pre, torch.zeros((), device=pre.device, dtype=torch.float64)) * live
    out = {k: torch.zeros_like(f[k[1:]]) for k in ("dx", "ddt", "dA", "dB", "dC")}
    G = torch.zeros_like(start)
    for t in reversed(range(length)):
        x, d, B, C = f["x"][:, t], delta[:, t], f["B"][:, t], f["C"][:, t]
        G = G + gy[:, t, :, None] * C[:, None]
        out["dC"][:, t] = (states[t] * gy[:, t, :, None]).sum(1)
        out["dB"][:, t] = (G * (d * x)[..., None]).sum(1)
        inner = (G * B[:, None]).sum(2)
        a = torch.exp(d[..., None] * f["A"])
        through = G * a * (states[t - 1] if t else start)
        out["dA"] += (through * d[..., None]).sum(0)
        out["ddt"][:, t] = (inner * x + (through * f["A"]).sum(2)) / (1 + torch.exp(-pre[:, t])) * live[:, t]
        out["dx"][:, t] = inner * d + gy[:, t] * f["D"]
        G = G * a
    return {"y": y * f["z"] * gate * live, "dx": out["dx"], "ddt": out["ddt"], "dA": out["dA"], "dB": out["dB"], "dC": out["dC"],
            "dD": (gy * f["x"]).sum((0, 1)), "dz": g * y * gate * (1 + f["z"] * (1 - gate)), "dbias": out["ddt"].sum((0, 1))}

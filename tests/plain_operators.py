"""Plain 64-bit forms of the prediction network's and the decoder's operators, on the CPU, for the tests.

Every function takes ``magnitude=True`` too: the same sums with the absolute value of every term, which bounds how far
rounding can carry a result (a sum of k terms, each off by a relative e, is off by at most (k u + e) times the sum of its
terms' magnitudes, u = 2^-24 for fp32 arithmetic)."""
import torch

U = 2.0 ** -24
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def f64(t):
    return None if t is None else t.detach().cpu().double()


def spacing(ref, dtype):
    """Half a step of ``dtype`` at ``ref``: what one rounding may be off by (fp16: also half its smallest subnormal)."""
    eps = torch.finfo(dtype).eps / 2
    return ref.abs() * eps + (2.0 ** -25 if dtype is torch.float16 else 1e-40)


def assert_within(got, ref, bound, what):
    """|got - ref| <= bound element by element; NaN and infinities in the same places."""
    got, ref = f64(got), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)]), what
    over = ((got - ref).abs() - bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, (what, float(over.max()), float((got - ref)[fine].abs().max()))


# ---- token embedding ---------------------------------------------------------------------------------------------------
def embedding(tokens, weight, scale, grad=None, padding=None, magnitude=False):
    w = weight.abs() if magnitude else weight
    flat = tokens.reshape(-1)
    ok = (flat >= 0) & (flat < weight.shape[0])
    out = w[flat.clamp(0, weight.shape[0] - 1)] * (abs(scale) if magnitude else scale)
    out[~ok] = float("nan")
    if grad is None:
        return out.reshape(*tokens.shape, -1)
    g = (grad.abs() if magnitude else grad).reshape(flat.numel(), -1)
    dweight = torch.zeros_like(w)
    for i in range(flat.numel()):
        if ok[i] and int(flat[i]) != (-1 if padding is None else padding):
            dweight[flat[i]] += g[i]
    return out.reshape(*tokens.shape, -1), dweight * (abs(scale) if magnitude else scale)


# ---- causal convolution --------------------------------------------------------------------------------------------------
def conv(x, w, b, init, lens, silu, gy=None, gfinal=None, magnitude=False):
    """-> dict(y, state[, dx, dw, db, dinit]); rows past the lengths are never looked at."""
    B, L, D = x.shape
    W = w.shape[1]
    m = (lambda t: t.abs()) if magnitude else (lambda t: t)
    y, state = torch.zeros(B, L, D, dtype=torch.float64), torch.zeros(B, W - 1, D, dtype=torch.float64)
    r = dict(y=y, state=state, dx=torch.zeros_like(y), dw=torch.zeros_like(w), db=torch.zeros(D, dtype=torch.float64),
             dinit=torch.zeros_like(state))
    for i in range(B):
        n = L if lens is None else int(lens[i])
        xe = torch.cat((torch.zeros(W - 1, D, dtype=torch.float64) if init is None else init[i], x[i, :n]))
        state[i] = xe[n:n + W - 1]
        p = (torch.stack([xe[k:k + n] * w[:, k] for k in range(W)]).sum(0) + (0 if b is None else b)) if n else torch.zeros(0, D).double()
        pm = (torch.stack([(xe[k:k + n] * w[:, k]).abs() for k in range(W)]).sum(0) + (0 if b is None else b.abs())) if n else p
        s = torch.sigmoid(p)
        y[i, :n] = (pm if magnitude else p * s) if silu else (pm if magnitude else p)
        dxe = torch.zeros(n + W - 1, D, dtype=torch.float64)
        if gfinal is not None:
            dxe[n:] += m(gfinal[i])
        if gy is not None:
            # silu' <= 1.1 and |silu''| <= 0.5: an error of p moves the gradient by half of it at most
            d = (1.1 + pm if magnitude else s + p * s * (1 - s)) if silu else torch.ones_like(p)
            gp = m(gy[i, :n]) * d
            for k in range(W):
                dxe[k:k + n] += gp * m(w[:, k])
                r["dw"][:, k] += (gp * m(xe[k:k + n])).sum(0)
            r["db"] += gp.sum(0)
        r["dx"][i, :n] = dxe[W - 1:]
        r["dinit"][i] = dxe[:W - 1]
    return r


# ---- selective scan ----------------------------------------------------------------------------------------------------------
def softplus(v):
    return torch.logaddexp(v, torch.zeros((), dtype=torch.float64))


def scan(x, dt, A, B, C, D=None, z=None, bias=None, init=None, lens=None, gy=None, gfinal=None, magnitude=False):
    """-> dict(y, state[, dx, ddt, dA, dB, dC, dD, dz, dbias, dinit])."""
    n_b, L, dim = x.shape
    N = A.shape[1]
    m = (lambda t: t.abs()) if magnitude else (lambda t: t)
    zeros = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
    skip, bias_ = zeros(dim) if D is None else D, zeros(dim) if bias is None else bias
    r = dict(y=zeros(n_b, L, dim), state=zeros(n_b, dim, N), dx=zeros(n_b, L, dim), ddt=zeros(n_b, L, dim), dA=zeros(dim, N),
             dB=zeros(n_b, L, N), dC=zeros(n_b, L, N), dD=zeros(dim), dz=zeros(n_b, L, dim), dbias=zeros(dim), dinit=zeros(n_b, dim, N))
    for i in range(n_b):
        n = L if lens is None else int(lens[i])
        h = zeros(dim, N) if init is None else m(init[i])
        states, pre = [h], dt[i, :n] + bias_
        delta, xs, Bs, Cs = softplus(pre), m(x[i, :n]), m(B[i, :n]), m(C[i, :n])
        if z is None:
            gate, dgate = torch.ones(n, dim, dtype=torch.float64), None
        else:
            zz, s = z[i, :n], torch.sigmoid(z[i, :n])
            gate, dgate = m(zz) * s, s + m(zz) * s * (1 - s)
        inner_y = zeros(n, dim)
        for t in range(n):
            h = torch.exp(delta[t, :, None] * A) * h + (delta[t] * xs[t])[:, None] * Bs[t]
            states.append(h)
            inner_y[t] = (h * Cs[t]).sum(1) + m(skip) * xs[t]
        r["y"][i, :n] = inner_y * gate
        r["state"][i] = h
        if gy is None and gfinal is None:
            continue
        g = zeros(n, dim) if gy is None else m(gy[i, :n])
        G = zeros(dim, N) if gfinal is None else m(gfinal[i])
        if z is not None:
            r["dz"][i, :n] = g * inner_y * dgate
        gi = g * gate
        r["dD"] += (gi * xs).sum(0)
        for t in reversed(range(n)):
            r["dC"][i, t] = (states[t + 1] * gi[t][:, None]).sum(0)
            G = G + gi[t][:, None] * Cs[t]
            r["dB"][i, t] = (G * (delta[t] * xs[t])[:, None]).sum(0)
            inner = (G * Bs[t]).sum(1)
            G = G * torch.exp(delta[t, :, None] * A)
            through = G * states[t]
            r["dA"] += through * delta[t][:, None]
            r["dx"][i, t] = inner * delta[t] + gi[t] * m(skip)
            r["ddt"][i, t] = (inner * xs[t] + (through * m(A)).sum(1)) * torch.sigmoid(pre[t])
        r["dbias"] += r["ddt"][i].sum(0)
        r["dinit"][i] = G
    return r


# ---- decoding rules ------------------------------------------------------------------------------------------------------------
def rules32(x, V, bias=None, allowed=None, history=None, history_lens=None, repetition=1.0, presence=0.0, frequency=0.0):
    """The rules in fp32, in the order that is documented: what the kernels have to give bit for bit.  ``allowed`` is bool."""
    v = x.detach().cpu().float().clone()
    rows = v.shape[0]
    contexts = max([t.shape[0] for t in (bias, allowed, history) if t is not None and t.dim() == 2] or [1])
    per = rows // contexts
    one = torch.ones((), dtype=torch.float32)
    for r in range(rows):
        c = r // per
        count = torch.zeros(V)
        if history is not None:
            n = history.shape[1] if history_lens is None else min(max(int(history_lens[c]), 0), history.shape[1])
            for t in history[c, :n].tolist():
                if 0 <= t < V:
                    count[t] += 1
        row = v[r]
        seen = count > 0
        row = torch.where(seen, torch.where(row > 0, row / (one * repetition), row * (one * repetition)), row)
        row = torch.where(seen, row - (one * frequency) * count, row)
        row = torch.where(seen, row - one * presence, row)
        if bias is not None:
            row = row + (bias[c] if bias.dim() == 2 else bias).cpu()
        if allowed is not None:
            row = row.masked_fill(~(allowed[c] if allowed.dim() == 2 else allowed).cpu(), float("-inf"))
        v[r] = row
    return v

"""GPU tests of causal_conv, selective_scan and their single-token forms against the plain 64-bit forms.

Tolerances (u = 2^-24).  Scan: softplus is within 6 u, a decay exp(delta A) within (7 |delta A| + 2) u and, since
x e^-x <= 1/e, counts for at most 5 u of what it passes on; a step adds two rounded operations; so a value that was carried
over L steps is within 8 (L + 1) u of its magnitude, the sum over N states adds N u, a gate z sigmoid(z) (4 + 2 |z|) u <= 16 u for the inputs here:
(8 (L + 1) + N + 32) u in all.  A gradient passes such a path twice, and a sum over n terms adds n u:
(16 (L + 1) + N + 64 + n) u.  Both times the magnitude that plain_operators computes, plus one rounding to the type."""
import pytest
import torch

import plain_operators as plain

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = plain.U


def lens_for(kind, B, L):
    if kind is None or torch.is_tensor(kind):
        return kind
    some = [L, 0, 1, max(1, L // 2), max(1, L - 1), (L + 2) // 3]
    return torch.tensor([some[i % len(some)] for i in range(B)], dtype=torch.int32)


def scan_inputs(B, L, D, N, dtype, seed=0, full=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    a = dict(x=r(B, L, D).to(dtype), dt=r(B, L, D).to(dtype), A=-torch.arange(1, N + 1).float() * (0.5 + torch.rand(D, 1, generator=g)),
             B=r(B, L, N).to(dtype), C=r(B, L, N).to(dtype))
    if full:
        a.update(D=r(D), z=r(B, L, D).to(dtype), bias=r(D) - 3, init=r(B, D, N))
    return a, dict(gy=r(B, L, D).to(dtype), gfinal=r(B, D, N))


def call_scan(a, lens):
    import rnnt_amd

    return rnnt_amd.selective_scan(a["x"], a["dt"], a["A"], a["B"], a["C"], D=a.get("D"), z=a.get("z"), dt_bias=a.get("bias"),
                                   initial_state=a.get("init"), lengths=None if lens is None else lens.to(DEV))


def check_scan(B, L, D, N, dtype, ragged, full, seed=0, poison=True, device_inputs=None, use_final=True):
    a, grads = scan_inputs(B, L, D, N, dtype, seed, full)
    lens = lens_for(ragged, B, L)
    ref_in = {k: v.double() for k, v in a.items()}
    ref_g = {k: v.double() for k, v in grads.items()}
    if not use_final:
        ref_g["gfinal"] = None
    if lens is not None and poison:  # what lies past a sequence's end is never looked at
        past = torch.arange(L)[None] >= lens[:, None]
        for k in ("x", "dt", "z", "B", "C"):
            if k in a:
                a[k][past] = float("nan")
        grads["gy"][past] = float("nan")
    dev = {k: v.to(DEV) for k, v in a.items()} if device_inputs is None else device_inputs(a)
    dev = {k: v.detach().requires_grad_(True) for k, v in dev.items()}
    y, state = call_scan(dev, lens)
    names = list(dev)
    outs, gos = ([y, state], [grads["gy"].to(DEV), grads["gfinal"].to(DEV)]) if use_final else ([y], [grads["gy"].to(DEV)])
    got = dict(zip(("d" + k for k in names), torch.autograd.grad(outs, [dev[k] for k in names], gos)))
    with torch.no_grad():
        y2, state2 = call_scan(dev, lens)
    assert torch.equal(y, y2) and torch.equal(state, state2)   # with and without the states kept
    lens_l = None if lens is None else lens.tolist()
    ref, mag = (plain.scan(**ref_in, lens=lens_l, **ref_g, magnitude=m) for m in (False, True))
    fwd, bwd = 8 * (L + 1) + N + 32, 16 * (L + 1) + N + 64
    plain.assert_within(y, ref["y"], fwd * U * mag["y"] + plain.spacing(ref["y"], dtype), "y")
    plain.assert_within(state, ref["state"], fwd * U * mag["state"] + 1e-40, "state")
    for k in names:
        n = {"B": D, "C": D, "A": B * L, "D": B * L, "bias": B * L}.get(k, 0)
        t = torch.float32 if k in ("A", "D", "bias", "init") else dtype
        assert got["d" + k].dtype is t
        plain.assert_within(got["d" + k], ref["d" + k], (bwd + n) * U * mag["d" + k] + plain.spacing(ref["d" + k], t), "d" + k)
    return dev, got


@pytest.mark.parametrize("dtype", plain.TYPES)
@pytest.mark.parametrize("B,L,D,N", [(1, 1, 1, 8), (2, 2, 3, 16), (3, 17, 64, 16), (2, 33, 70, 8), (6, 16, 65, 16), (1, 130, 66, 32),
                                     (2, 5, 129, 32)])
def test_scan_against_plain(dtype, B, L, D, N):
    check_scan(B, L, D, N, dtype, ragged=B > 1, full=True, seed=L)


@pytest.mark.parametrize("dtype", plain.TYPES)
@pytest.mark.parametrize("N", [8, 16, 32])
def test_scan_over_several_segments(dtype, N):
    check_scan(3, 275, 20, N, dtype, ragged=True, full=True, seed=N)
    check_scan(1, 257, 65, N, dtype, ragged=None, full=False, seed=N)


@pytest.mark.parametrize("keep", ["none", "D", "z", "bias", "init"])
def test_scan_with_each_optional_argument_alone(keep):
    a, grads = scan_inputs(2, 19, 10, 16, torch.float32, seed=1)
    a = {k: v for k, v in a.items() if k in ("x", "dt", "A", "B", "C", keep)}
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in a.items()}
    y, state = call_scan(dev, None)
    got = torch.autograd.grad([y, state], list(dev.values()), [grads["gy"].to(DEV), grads["gfinal"].to(DEV)])
    ref, mag = (plain.scan(**{k: v.double() for k, v in a.items()}, gy=grads["gy"].double(), gfinal=grads["gfinal"].double(), magnitude=m)
                for m in (False, True))
    plain.assert_within(y, ref["y"], 220 * U * mag["y"], "y")
    for k, v in zip(dev, got):
        plain.assert_within(v, ref["d" + k], 500 * U * mag["d" + k] + 1e-40, k)


def test_scan_gradient_of_one_result_only():
    check_scan(2, 20, 33, 16, torch.float32, ragged=True, full=True, use_final=False)
    a, grads = scan_inputs(2, 20, 12, 16, torch.float32, seed=9)
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in a.items()}
    _, state = call_scan(dev, None)
    got = torch.autograd.grad(state, [dev[k] for k in ("x", "init", "A")], grads["gfinal"].to(DEV))
    ref, mag = (plain.scan(**{k: v.double() for k, v in a.items()}, gfinal=grads["gfinal"].double(), magnitude=m) for m in (False, True))
    for k, v in zip(("x", "init", "A"), got):
        plain.assert_within(v, ref["d" + k], 500 * U * mag["d" + k] + 1e-40, k)


@pytest.mark.parametrize("dtype", plain.TYPES)
@pytest.mark.parametrize("shift", [0, 1, 2, 5])
def test_scan_layouts(dtype, shift):
    """x and z as halves of one projection, B and C as parts of another that start off every alignment, and the state rows
    of odd length that put every other row on an odd element."""
    def apart(a):
        B, L, D = a["x"].shape
        N = a["A"].shape[1]
        xz = torch.full((B, L, 2 * D + shift), float("nan"), dtype=dtype)
        xz[..., shift:shift + D], xz[..., shift + D:] = a["x"], a["z"]
        bc = torch.full((L, B, 2 * N + 5 + shift), float("nan"), dtype=dtype)      # time first, too
        bc[..., shift:shift + N], bc[..., shift + N + 1:shift + 2 * N + 1] = a["B"].transpose(0, 1), a["C"].transpose(0, 1)
        xz, bc = xz.to(DEV), bc.to(DEV).transpose(0, 1)
        dev = {k: v.to(DEV) for k, v in a.items()}
        dev.update(x=xz[..., shift:shift + D], z=xz[..., shift + D:], B=bc[..., shift:shift + N], C=bc[..., shift + N + 1:shift + 2 * N + 1],
                   dt=dev["dt"].transpose(1, 2).contiguous().transpose(1, 2))       # channels apart: laid out by the call
        return dev
    check_scan(3, 21, 37, 16, dtype, ragged=True, full=True, seed=shift, device_inputs=apart)


def test_scan_broadcast_inputs():
    """B of one sequence expanded over the batch: its gradient is the sum over the sequences."""
    a, grads = scan_inputs(3, 9, 8, 16, torch.float32, seed=4)
    one = a["B"][:1].to(DEV).requires_grad_(True)
    dev = {k: v.to(DEV) for k, v in a.items()}
    y, _ = call_scan({**dev, "B": one.expand(3, 9, 16)}, None)
    got, = torch.autograd.grad(y, one, grads["gy"].to(DEV))
    whole = {**{k: v.double() for k, v in a.items()}, "B": a["B"][:1].double().expand(3, 9, 16)}
    ref, mag = (plain.scan(**whole, gy=grads["gy"].double(), magnitude=m) for m in (False, True))
    plain.assert_within(got, ref["dB"].sum(0, keepdim=True), 300 * U * mag["dB"].sum(0, keepdim=True), "dB")


def test_scan_extreme_steps():
    """dt far to both sides (delta 0 and huge), A of 0 and of huge rates, and infinities and NaN that stay in their sequence."""
    a, _ = scan_inputs(4, 6, 8, 8, torch.float32, seed=3)
    a["dt"][0, :, 0], a["dt"][0, :, 1], a["dt"][0, :, 2] = -200.0, 80.0, -float("inf")
    a["A"][3], a["A"][4] = 0.0, -1e6
    a["x"][2, 3, 5] = float("nan")
    a["x"][3, 2, 6] = float("inf")
    y, state = call_scan({k: v.to(DEV) for k, v in a.items()}, None)
    ref, mag = (plain.scan(**{k: v.double() for k, v in a.items()}, magnitude=m) for m in (False, True))
    y, state = y.cpu(), state.cpu()
    assert torch.isnan(y[2, 3:, 5]).all() and torch.isfinite(y[2, :3]).all() and torch.isfinite(y[2, :, :5]).all()
    assert torch.isfinite(y[:2]).all()
    plain.assert_within(y[:2], ref["y"][:2], 200 * U * mag["y"][:2] + 1e-37, "y")
    plain.assert_within(state[:2], ref["state"][:2], 200 * U * mag["state"][:2] + 1e-37, "state")
    assert not torch.isfinite(y[3, 2:, 6]).any()


def test_prompt_then_tokens_is_the_whole_sequence():
    """A prompt in two calls and then tokens one by one, through convolution and scan, against one call over everything."""
    import rnnt_amd

    g = torch.Generator().manual_seed(2)
    B, L, D, N, W = 3, 40, 72, 16, 4
    a, _ = scan_inputs(B, L, D, N, torch.float32, seed=2)
    w, b = torch.randn(D, W, generator=g).to(DEV), torch.randn(D, generator=g).to(DEV)
    a = {k: v.to(DEV) for k, v in a.items()}

    def layer(lo, hi, conv_state, scan_state, step=False):
        cut = {k: (a[k][:, lo] if step else a[k][:, lo:hi]) for k in ("x", "dt", "B", "C", "z")}
        if step:
            x, conv_state = rnnt_amd.causal_conv_step(cut["x"], conv_state, w, b)
            y, scan_state = rnnt_amd.selective_scan_step(x, cut["dt"], a["A"], cut["B"], cut["C"], scan_state, D=a["D"], z=cut["z"], dt_bias=a["bias"])
            return y[:, None], conv_state, scan_state
        x, conv_state = rnnt_amd.causal_conv(cut["x"], w, b, initial_state=conv_state)
        y, scan_state = rnnt_amd.selective_scan(x, cut["dt"], a["A"], cut["B"], cut["C"], D=a["D"], z=cut["z"], dt_bias=a["bias"],
                                                initial_state=scan_state)
        return y, conv_state, scan_state

    with torch.no_grad():
        whole, conv_all, scan_all = layer(0, L, None, a["init"])
        parts, conv, scan = [], None, a["init"]
        for lo, hi in ((0, 2), (2, 30)):
            y, conv, scan = layer(lo, hi, conv, scan)
            parts.append(y)
        for t in range(30, L):
            y, conv, scan = layer(t, t + 1, conv, scan, step=True)
            parts.append(y)
    assert torch.equal(conv, conv_all)
    # both sides compute the same sums, each within 8 (L + 1) u + ... of them
    ref = plain.conv(plain.f64(a["x"]), plain.f64(w), plain.f64(b), None, None, True)["y"].float()
    mag = plain.scan(**{**{k: plain.f64(v) for k, v in a.items()}, "x": ref.double()}, magnitude=True)
    limit = 2 * (8 * (L + 1) + N + 64) * U
    plain.assert_within(torch.cat(parts, 1), plain.f64(whole), limit * mag["y"] + 1e-5 * U, "y")
    plain.assert_within(scan, plain.f64(scan_all), limit * mag["state"] + 1e-5 * U, "state")


@pytest.mark.parametrize("dtype", plain.TYPES)
@pytest.mark.parametrize("B,D,N", [(1, 1, 8), (1, 7, 16), (3, 64, 32), (5, 130, 16), (2, 66, 8), (257, 9, 16)])
def test_scan_step(dtype, B, D, N):
    import rnnt_amd

    a, _ = scan_inputs(B, 1, D, N, dtype, seed=D)
    ref, mag = (plain.scan(**{k: v.double() for k, v in a.items()}, magnitude=m) for m in (False, True))
    dev = {k: v.to(DEV) for k, v in a.items()}
    row = {k: dev[k][:, 0] for k in ("x", "dt", "B", "C", "z")}
    before = dev["init"].clone()
    args = (row["x"], row["dt"], dev["A"], row["B"], row["C"])
    y, state = rnnt_amd.selective_scan_step(*args, dev["init"], D=dev["D"], z=row["z"], dt_bias=dev["bias"])
    assert torch.equal(dev["init"], before)
    plain.assert_within(y, ref["y"][:, 0], (N + 48) * U * mag["y"][:, 0] + plain.spacing(ref["y"][:, 0], dtype), "y")
    plain.assert_within(state, ref["state"], 48 * U * mag["state"] + 1e-40, "state")
    y2, same = rnnt_amd.selective_scan_step(*args, dev["init"], D=dev["D"], z=row["z"], dt_bias=dev["bias"], state_out=dev["init"])
    assert same.data_ptr() == dev["init"].data_ptr() and torch.equal(dev["init"], state) and torch.equal(y, y2)
    y3, _ = rnnt_amd.selective_scan_step(*args, before)           # without D, z, dt_bias
    bare = plain.scan(*(a[k].double() for k in ("x", "dt", "A", "B", "C")), init=a["init"].double())
    bare_mag = plain.scan(*(a[k].double() for k in ("x", "dt", "A", "B", "C")), init=a["init"].double(), magnitude=True)
    plain.assert_within(y3, bare["y"][:, 0], (N + 48) * U * bare_mag["y"][:, 0] + plain.spacing(bare["y"][:, 0], dtype), "y bare")


# ---- convolution -------------------------------------------------------------------------------------------------------------
# p is a sum of W + 1 products; y = p sigmoid(p) moves by at most 1.1 of p's error and is off by (4 + 2 |p|) u itself
def conv_inputs(B, L, D, W, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    a = dict(x=r(B, L, D).to(dtype), w=r(D, W) / W ** 0.5, b=r(D), init=r(B, W - 1, D).to(dtype))
    return a, r(B, L, D).to(dtype), r(B, W - 1, D).to(dtype)


def check_conv(B, L, D, W, dtype, ragged, silu=True, state=True, bias=True, seed=0, layout=None):
    import rnnt_amd

    a, gy, gf = conv_inputs(B, L, D, W, dtype, seed)
    lens = lens_for(ragged, B, L)
    c = [a["x"].double(), a["w"].double(), a["b"].double() if bias else None, a["init"].double() if state else None]
    ref, mag = (plain.conv(*c, None if lens is None else lens.tolist(), silu, gy.double(), gf.double(), magnitude=m) for m in (False, True))
    if lens is not None:
        past = torch.arange(L)[None] >= lens[:, None]
        a["x"][past], gy[past] = float("nan"), float("nan")
    dev = {k: v.to(DEV) for k, v in a.items()}
    if layout is not None:
        dev["x"] = layout(dev["x"])
    dev = {k: v.detach().requires_grad_(True) for k, v in dev.items()}
    used = [dev["x"], dev["w"]] + ([dev["b"]] if bias else []) + ([dev["init"]] if state else [])
    y, final = rnnt_amd.causal_conv(dev["x"], dev["w"], dev["b"] if bias else None, dev["init"] if state else None,
                                    None if lens is None else lens.to(DEV), "silu" if silu else None)
    got = torch.autograd.grad([y, final], used, [gy.to(DEV), gf.to(DEV)])
    limit = (8 * W + 48) * U
    plain.assert_within(y, ref["y"], limit * mag["y"] + plain.spacing(ref["y"], dtype), "y")
    assert torch.equal(final.cpu(), ref["state"].to(dtype))
    for k, v in zip(["dx", "dw"] + (["db"] if bias else []) + (["dinit"] if state else []), got):
        n = B * L if k in ("dw", "db") else 0
        plain.assert_within(v, ref[k], (limit + n * U) * mag[k] + plain.spacing(ref[k], v.dtype), k)


@pytest.mark.parametrize("dtype", plain.TYPES)
@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("B,L,D", [(1, 1, 1), (2, 2, 8), (6, 3, 5), (6, 32, 24), (6, 33, 257), (2, 150, 16)])
def test_conv_against_plain(dtype, W, B, L, D):
    check_conv(B, L, D, W, dtype, ragged=B > 1, seed=L + W)


@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("state", [True, False])
@pytest.mark.parametrize("bias", [True, False])
def test_conv_options(silu, state, bias):
    check_conv(6, 20, 40, 4, torch.float32, True, silu, state, bias)


@pytest.mark.parametrize("W", [2, 3, 4])
@pytest.mark.parametrize("state", [True, False])
def test_conv_ends_around_blocks_and_runs(W, state):
    """Sequences that end in, before and behind blocks of 8 steps and runs of 32 and 64, at every distance up to the filter's width."""
    lens = torch.tensor([*range(13), *range(28, 37), *range(60, 76), *range(124, 141)], dtype=torch.int32)
    check_conv(len(lens), 140, 5, W, torch.float32, lens, state=state, seed=W)


def test_conv_layouts():
    half = lambda x: torch.cat((torch.full_like(x, float("nan")), x), 2)[..., x.shape[2]:]  # noqa: E731
    odd = lambda x: torch.cat((x[..., :1], x, x[..., :2]), 2)[..., 1:1 + x.shape[2]]  # noqa: E731
    time_first = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    apart = lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    for layout in (half, odd, time_first, apart):
        for dtype in plain.TYPES:
            check_conv(6, 37, 32, 4, dtype, True, layout=layout)


@pytest.mark.parametrize("dtype", plain.TYPES)
@pytest.mark.parametrize("B,D,W", [(1, 1, 2), (3, 65, 4), (300, 8, 3)])
def test_conv_step(dtype, B, D, W):
    import rnnt_amd

    a, _, _ = conv_inputs(B, 1, D, W, dtype, seed=D)
    ref, mag = (plain.conv(a["x"].double(), a["w"].double(), a["b"].double(), a["init"].double(), None, True, magnitude=m) for m in (False, True))
    dev = {k: v.to(DEV) for k, v in a.items()}
    before = dev["init"].clone()
    y, state = rnnt_amd.causal_conv_step(dev["x"][:, 0], dev["init"], dev["w"], dev["b"])
    assert torch.equal(dev["init"], before) and torch.equal(state.cpu(), ref["state"].to(dtype))
    plain.assert_within(y, ref["y"][:, 0], (8 * W + 48) * U * mag["y"][:, 0] + plain.spacing(ref["y"][:, 0], dtype), "y")
    y2, same = rnnt_amd.causal_conv_step(dev["x"][:, 0], dev["init"], dev["w"], dev["b"], state_out=dev["init"])
    assert same.data_ptr() == dev["init"].data_ptr() and torch.equal(dev["init"], state) and torch.equal(y, y2)


def test_offsets_past_32_bits():
    """Two sequences whose rows lie more than 2^32 bytes apart, and steps that far apart: the results of the packed ones."""
    import rnnt_amd

    far = 1 << 31                                           # elements of bf16: 4 GiB
    pool = torch.empty(far + (1 << 20), dtype=torch.bfloat16, device=DEV)
    a, grads = scan_inputs(2, 20, 64, 16, torch.bfloat16, seed=6)
    dev = {k: v.to(DEV) for k, v in a.items()}
    gy = grads["gy"].to(DEV)
    w = torch.randn(64, 4, device=DEV)

    def results(x, B, gy):
        leaves = [t.detach().requires_grad_(True) for t in (x, B)]
        y, state = call_scan({**dev, "x": leaves[0], "B": leaves[1]}, None)
        out = (y, state, *torch.autograd.grad(y, leaves, gy))
        y, state = rnnt_amd.causal_conv(leaves[0], w)
        return out + (y, state, torch.autograd.grad(y, leaves[0], gy)[0])

    want = results(dev["x"], dev["B"], gy)
    views = []
    for k, (t, at) in enumerate(((dev["x"], 0), (dev["B"], 4096), (gy, 8192))):
        v = pool.as_strided(t.shape, (far, t.shape[2], 1), at)
        v.copy_(t)
        views.append(v)
    for p, q in zip(want, results(*views)):
        assert torch.equal(p, q)
    one = {k: (v[:1, :2] if v.dim() == 3 and k != "init" else v) for k, v in dev.items()}
    one["init"] = dev["init"][:1]
    x_far = pool.as_strided((1, 2, 64), (64, far, 1), 0)     # two steps of one sequence
    x_far.copy_(one["x"])
    assert all(torch.equal(p, q) for p, q in zip(call_scan(one, None), call_scan({**one, "x": x_far}, None)))
    assert torch.equal(rnnt_amd.causal_conv(one["x"], w)[0], rnnt_amd.causal_conv(x_far, w)[0])


# ---- how they are called -----------------------------------------------------------------------------------------------------
def test_same_bits_every_time_and_on_another_stream():
    a, grads = scan_inputs(3, 300, 96, 16, torch.bfloat16, seed=7)
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in a.items()}
    gy = grads["gy"].to(DEV)
    torch.cuda.synchronize()
    side, first = torch.cuda.Stream(), None
    for i in range(4):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            y, _ = call_scan(dev, None)
            got = (y, *torch.autograd.grad(y, list(dev.values()), gy))
        torch.cuda.synchronize()
        first = first or got
        assert all(torch.equal(p, q) for p, q in zip(first, got))


def test_captured_and_replayed():
    """Steps, prompts and a training pass in HIP graphs (two graphs, each with its own buffers), replayed in turn with eager
    calls between."""
    import rnnt_amd

    a, grads = scan_inputs(2, 150, 64, 16, torch.float32, seed=5)
    dev = {k: v.to(DEV) for k, v in a.items()}
    leaves = {k: v.detach().clone().requires_grad_(True) for k, v in dev.items()}
    gy = grads["gy"].to(DEV)
    cut = {k: dev[k][:, 0] for k in ("x", "dt", "B", "C", "z")}
    w = torch.randn(64, 4, device=DEV)
    conv0 = torch.randn(2, 3, 64, device=DEV)

    def decode():
        x, conv = rnnt_amd.causal_conv_step(cut["x"], conv0, w)
        y, state = rnnt_amd.selective_scan_step(x, cut["dt"], dev["A"], cut["B"], cut["C"], dev["init"], D=dev["D"], z=cut["z"], dt_bias=dev["bias"])
        with torch.no_grad():
            return (y, conv, state, *call_scan(dev, None))

    def train():
        x, _ = rnnt_amd.causal_conv(leaves["x"], w)
        y, _ = call_scan({**leaves, "x": x}, None)
        return (y, *torch.autograd.grad(y, list(leaves.values()), gy))

    graphs = []
    for fn in (decode, train):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fn()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fn()
        graphs.append((graph, out, fn))
    for seed in range(3):
        fresh, _ = scan_inputs(2, 150, 64, 16, torch.float32, seed=50 + seed)
        with torch.no_grad():
            for k in dev:
                dev[k].copy_(fresh[k])
                leaves[k].copy_(fresh[k])
        for graph, out, fn in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, fn()))


def test_refusals_on_the_device():
    import rnnt_amd

    a = {k: v.to(DEV) for k, v in scan_inputs(2, 3, 8, 8, torch.float32)[0].items()}
    leaf = a["x"].requires_grad_(True)
    y, _ = call_scan(a, None)
    g, = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        g.sum().backward()
    row = [a[k][:, 0] for k in ("x", "dt")] + [a["A"]] + [a[k][:, 0] for k in ("B", "C")]
    with pytest.raises(RuntimeError, match="no backward"):
        rnnt_amd.selective_scan_step(*row, a["init"])
    with torch.no_grad():
        pool = torch.zeros(2 * 8 * 8 + 8, device=DEV)
        state = pool[:128].view(2, 8, 8)
        with pytest.raises(ValueError, match="overlap"):
            rnnt_amd.selective_scan_step(*row, state, state_out=pool[8:].view(2, 8, 8))
        with pytest.raises(ValueError, match="state_out must be contiguous"):
            rnnt_amd.selective_scan_step(*row, state, state_out=torch.zeros(2, 8, 9, device=DEV)[..., :8])
        with pytest.raises(TypeError, match="state_out must have the state's type"):
            rnnt_amd.selective_scan_step(*row, state, state_out=state.half())
        with pytest.raises(RuntimeError, match="state must be on"):
            rnnt_amd.selective_scan_step(*row, state.cpu())
        with pytest.raises(RuntimeError, match="lengths must be on"):
            rnnt_amd.selective_scan(a["x"], a["dt"], a["A"], a["B"], a["C"], lengths=torch.zeros(2, dtype=torch.int32))


def test_scan_of_growing_states_over_segments():
    """A > 0: over 16 steps the states grow by e^96, more than fp32 holds, from 1e-30; and zeros stay zeros.  The exponent of 96 is off by
    7 * 96 u from its steps and, where a segment's steps are added up first, by 16 u of it; 96 steps of 3 roundings: 2500 u of a
    value that is carried once, twice that for products of a state and a gradient."""
    L, D, N = 96, 4, 8
    a, grads = scan_inputs(1, L, D, N, torch.float32, seed=21)
    a["A"].fill_(1.0)
    a["bias"].zero_()
    a["dt"].fill_(-200.0)
    a["dt"][:, 32:48] = 6.0
    a["x"].zero_()
    a["init"] *= 1e-30
    a["init"][:, 1] = 0.0
    grads = {k: v * 1e-30 for k, v in grads.items()}
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in a.items()}
    y, state = call_scan(dev, None)
    got = torch.autograd.grad([y, state], list(dev.values()), [grads["gy"].to(DEV), grads["gfinal"].to(DEV)])
    ref, mag = (plain.scan(**{k: v.double() for k, v in a.items()}, lens=None, gy=grads["gy"].double(), gfinal=grads["gfinal"].double(),
                           magnitude=m) for m in (False, True))
    assert float(ref["state"].abs().max()) > 1e10 and torch.count_nonzero(state[:, 1]) == 0
    plain.assert_within(y, ref["y"], 2500 * U * mag["y"] + 1e-37, "y")
    plain.assert_within(state, ref["state"], 2500 * U * mag["state"] + 1e-37, "state")
    for k, g in zip(dev, got):
        plain.assert_within(g, ref["d" + k], 5000 * U * mag["d" + k] + 1e-37, "d" + k)


def test_results_in_the_callers_buffer():
    """Nothing that a step reads may lie in it, and autograd learns that it changed."""
    import rnnt_amd

    a = {k: v.to(DEV) for k, v in scan_inputs(2, 1, 8, 8, torch.float32)[0].items()}
    row = [a[k][:, 0] for k in ("x", "dt")] + [a["A"]] + [a[k][:, 0] for k in ("B", "C")]
    kept = a["init"].clone().requires_grad_(True) * 1
    z = kept.square().sum()
    with torch.no_grad():
        for i in (0, 1, 2, 3, 4):
            out = torch.zeros(2, 8, 8, device=DEV)
            args = list(row)
            args[i] = out.view(-1)[-args[i].numel():].view(args[i].shape)
            with pytest.raises(ValueError, match="state_out must not overlap another argument"):
                rnnt_amd.selective_scan_step(*args, a["init"], state_out=out)
        conv = torch.zeros(2, 3, 8, device=DEV)
        w = torch.randn(8, 4, device=DEV)
        with pytest.raises(ValueError, match="state_out must not overlap another argument"):
            rnnt_amd.causal_conv_step(conv[:, 1], torch.zeros(2, 3, 8, device=DEV), w, state_out=conv)
        want = rnnt_amd.selective_scan_step(*row, kept.clone())[1]
        _, state = rnnt_amd.selective_scan_step(*row, kept, state_out=kept)
        assert state.data_ptr() == kept.data_ptr() and torch.equal(kept, want)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        z.backward()


def test_backward_twice_gives_the_same_bits():
    import rnnt_amd

    a, grads = scan_inputs(2, 150, 64, 16, torch.bfloat16, seed=8)
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in a.items()}
    w = torch.randn(64, 4, device=DEV, requires_grad=True)
    x, _ = rnnt_amd.causal_conv(dev["x"], w)
    y, _ = call_scan({**dev, "x": x}, None)
    leaves = [*dev.values(), w]
    first, again = (torch.autograd.grad(y, leaves, grads["gy"].to(DEV), retain_graph=True) for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(first, again))

"""GPU tests of rnnt_amd.token_embedding / TokenEmbedding against the plain 64-bit form (plain_operators.py).

Tolerances: the forward rounds scale * w to fp32 and then to the type; the backward adds k values in fp32 (each addition
off by u times the partial sum, so at most k u times the sum of magnitudes), scales and rounds once."""
import pytest
import torch

import plain_operators as plain

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = plain.U


def make(n, V, D, dtype, seed=0, index=torch.int64, skew=3.0):
    g = torch.Generator().manual_seed(seed)
    tokens = (torch.rand(n, generator=g).pow(skew) * V).long().clamp(max=V - 1).to(index)
    return tokens, torch.randn(V, D, generator=g).to(dtype), torch.randn(*tokens.shape, D, generator=g).to(dtype)


def check(tokens, weight, grad, scale, padding, weight_dev=None, grad_dev=None):
    import rnnt_amd

    scale32 = float(torch.tensor(scale, dtype=torch.float32))
    w = (weight.to(DEV) if weight_dev is None else weight_dev).detach().requires_grad_(True)
    out = rnnt_amd.token_embedding(tokens.to(DEV), w, scale, padding)
    dw, = torch.autograd.grad(out, w, grad.to(DEV) if grad_dev is None else grad_dev)
    assert out.dtype is weight.dtype and dw.dtype is weight.dtype and out.shape == (*tokens.shape, weight.shape[1])
    ref, dref = plain.embedding(tokens, weight.double(), scale32, grad.double(), padding)
    _, mag = plain.embedding(tokens, weight.double(), scale32, grad.double(), padding, magnitude=True)
    plain.assert_within(out, ref, 2 * U * ref.abs() + plain.spacing(ref, weight.dtype), "out")
    flat = tokens.reshape(-1).long()
    k = torch.bincount(flat[(flat >= 0) & (flat < weight.shape[0])], minlength=weight.shape[0]).double()[:, None]
    plain.assert_within(dw, dref, (k + 2) * U * mag + plain.spacing(dref, weight.dtype), "dweight")
    return out.detach(), dw


@pytest.mark.parametrize("dtype", plain.TYPES)
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 7, 8), (3, 5, 64), (33, 9, 24), (65, 300, 129), (1312, 4232, 64), (700, 40, 520),
                                   (4096, 37, 8), (4097, 37, 8), (9000, 70000, 8), (5000, 256, 16), (5000, 255, 16)])
def test_against_plain(dtype, n, V, D):
    check(*make(n, V, D, dtype, seed=n + V), scale=1.0 if n % 2 else 22.627417, padding=None)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("n", [50, 6000])
def test_padding_and_tokens_outside_the_vocabulary(index, n):
    tokens, weight, grad = make(n, 30, 16, torch.float32, seed=2, index=index)
    tokens[::3] = 4                       # a frequent token that is the padding row
    tokens[1], tokens[2], tokens[5] = -1, 30, torch.iinfo(index).max
    if index is torch.int64:
        tokens[7] = (1 << 32) + 3         # its low half is a token
    _, dw = check(tokens, weight, grad, 2.0, 4)
    assert torch.count_nonzero(dw[4]) == 0
    check(tokens, weight, grad, 2.0, None)


def test_one_token_everywhere_and_no_token_of_a_row():
    for n in (31, 32, 33, 64, 4095, 12345):      # pieces that end with the run, inside it and after it
        tokens, weight, grad = make(n, 50, 32, torch.bfloat16, seed=n)
        tokens[:] = 49
        _, dw = check(tokens, weight, grad, 0.5, None)
        assert torch.count_nonzero(dw[:49]) == 0


@pytest.mark.parametrize("n,V", [(2048, 128), (2048, 127), (2049, 4000), (700, 50), (129, 1000)])
def test_frequent_tokens_in_short_sequences(n, V):
    """Both sides of the rule that picks the unsorted kernel (2048 positions, 16 to a row), with one row of most of them and
    two of more than a wave sums alone."""
    tokens, weight, grad = make(n, V, 72, torch.float32, seed=n)
    tokens[: n // 2] = V - 1
    tokens[n // 2::3] = 0
    check(tokens, weight, grad, 1.25, None)
    check(tokens, weight.bfloat16(), grad.bfloat16(), 1.25, 0)
    wide, more = torch.randn(V, 600, generator=torch.Generator().manual_seed(1)), torch.randn(n, 600, generator=torch.Generator().manual_seed(2))
    check(tokens, wide, more, 1.0, None)


def test_layouts():
    """Rows of the weight and of the gradient that lie apart, start off 16 bytes, repeat, or belong to a broadcast gradient."""
    tokens, weight, grad = make(90, 20, 24, torch.float16, seed=8)
    wide = torch.zeros(20, 40, dtype=torch.float16)
    wide[:, 3:27] = weight
    check(tokens, weight, grad, 3.0, 0, weight_dev=wide.to(DEV)[:, 3:27])
    check(tokens, weight.t().contiguous().t(), grad, 3.0, 0, weight_dev=weight.t().contiguous().to(DEV).t())
    check(tokens, weight, grad, 1.0, None, grad_dev=torch.cat((grad, grad), 1).to(DEV)[:, 24:])
    same = grad[:1].expand(90, 24)
    check(tokens, weight, same, 1.0, None, grad_dev=grad[:1].to(DEV).expand(90, 24))
    two = tokens.reshape(9, 10).t()
    check(two, weight, grad.reshape(10, 9, 24), 1.0, None)


def test_same_bits_every_time_and_on_another_stream():
    import rnnt_amd

    tokens, weight, grad = (t.to(DEV) for t in make(20000, 16384, 64, torch.float32, seed=4))
    w = weight.requires_grad_(True)
    first = torch.autograd.grad(rnnt_amd.token_embedding(tokens, w), w, grad)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for i in range(4):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            again = torch.autograd.grad(rnnt_amd.token_embedding(tokens, w), w, grad)[0]
        torch.cuda.synchronize()
        assert torch.equal(first, again)


def test_captured_and_replayed():
    """Forward and backward entry points in a HIP graph, replayed with new tokens between eager calls."""
    import rnnt_amd

    for n in (500, 5000):
        tokens, weight, grad = (t.to(DEV) for t in make(n, 300, 40, torch.float32, seed=n))
        w = weight.requires_grad_(True)

        def step():
            out = rnnt_amd.token_embedding(tokens, w, 1.5)
            return out, torch.autograd.grad(out, w, grad)[0]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, dw = step()
        for seed in range(3):
            tokens.copy_(make(n, 300, 40, torch.float32, seed=100 + seed)[0])
            graph.replay()
            torch.cuda.synchronize()
            eager = step()
            assert torch.equal(out, eager[0]) and torch.equal(dw, eager[1])


def test_module_is_a_drop_in_and_second_derivatives_raise():
    import rnnt_amd

    theirs = torch.nn.Embedding(11, 6, padding_idx=0)
    ours = rnnt_amd.TokenEmbedding(11, 6, padding_idx=0)
    ours.load_state_dict(theirs.state_dict())
    theirs, ours = theirs.to(DEV), ours.to(DEV)
    tokens = torch.tensor([[0, 3, 3], [10, 0, 1]], device=DEV)
    a, b = theirs(tokens), ours(tokens)
    assert torch.equal(a, b)
    a.square().sum().backward()
    b.square().sum().backward()
    torch.testing.assert_close(theirs.weight.grad, ours.weight.grad, rtol=4 * U, atol=0)
    assert rnnt_amd.TokenEmbedding(4, 16, scale="sqrt").scale == 4.0
    g, = torch.autograd.grad(ours(tokens).square().sum(), ours.weight, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        g.sum().backward()


def test_tensors_elsewhere_are_refused():
    import rnnt_amd

    with pytest.raises(RuntimeError, match="tokens must be on"):
        rnnt_amd.token_embedding(torch.zeros(2, dtype=torch.int64), torch.zeros(3, 4, device=DEV))


def test_offsets_past_32_bits():
    """Weight rows, and rows of the gradient, 4 GiB apart."""
    import rnnt_amd

    tokens, weight, grad = make(300, 2, 64, torch.bfloat16, seed=3)
    far = 1 << 31
    pool = torch.empty(far + 4096, dtype=torch.bfloat16, device=DEV)
    w = pool.as_strided((2, 64), (far, 1), 0)
    w.copy_(weight)
    check(tokens, weight, grad, 2.0, None, weight_dev=w)
    two = pool.as_strided((2, 64), (far, 1), 1024)
    two.copy_(grad[:2])
    check(tokens[:2], weight, grad[:2], 2.0, None, grad_dev=two)


@pytest.mark.parametrize("n,V", [((3 << 17) - 1, 300), (3 << 17, 300), (500_001, 70_000), ((1 << 21) + 77, 65_537)])
def test_many_positions(n, V):
    """Both ways of the sort: workgroups that add up the counts before them, and counts summed by a launch of their own."""
    check(*make(n, V, 4, torch.float32, seed=n), scale=1.0, padding=0)


def test_more_rows_than_one_launch_takes():
    """A lane per element and 64 lanes to a row: 2^25 rows a launch."""
    import rnnt_amd

    n, g = (1 << 25) + 3, torch.Generator(device=DEV).manual_seed(4)
    weight = torch.randn(11, 33, generator=g, device=DEV).bfloat16()
    for index in (torch.int32, torch.int64):
        tokens = torch.randint(0, 11, (n,), generator=g, device=DEV, dtype=index)
        out = rnnt_amd.token_embedding(tokens, weight, 2.0)
        for part in (slice(0, 1000), slice(n - 1000, n)):
            assert torch.equal(out[part], weight[tokens[part].long()] * 2)      # (times 2: exact)
        assert torch.equal(out.view(torch.int16).sum(1, dtype=torch.int64),
                           (weight * 2).view(torch.int16).sum(1, dtype=torch.int64)[tokens.long()])


def test_backward_twice_and_after_the_tokens_changed():
    import rnnt_amd

    tokens, weight, grad = (t.to(DEV) for t in make(300, 20, 8, torch.float32))
    w = weight.requires_grad_(True)
    out = rnnt_amd.token_embedding(tokens, w)
    first, again = (torch.autograd.grad(out, w, grad, retain_graph=True)[0] for _ in range(2))
    assert torch.equal(first, again)
    tokens.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(out, w, grad)

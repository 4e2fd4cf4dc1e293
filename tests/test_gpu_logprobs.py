"""Log-probabilities of tokens without the logits (``kernels/logprobs.py``) against 64 bits.

Bound of the results where the logits are exact: an exponent (z - m) log2 e is rounded twice, 2^-23 of its size; weighted
with the probabilities that size is the entropy at most, log2 of the vocabulary, below 18 here; sums of exponentials
are of 32 partial sums at most along any path and two roundings at each joining; the exponential, the logarithm and the last sums add
a few units of the results.  2^-24 (120 + 4 |result| + 4 |lse|) covers them.  Where the logits are fp32 sums of K
products, an error of each, K 2^-24 of the sum of the products' sizes at most, passes on once to lse and once more to the target."""
import math

import pytest
import torch

from kernels import _native
from kernels.logprobs import token_logprobs

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _whole(g, t, v, k, dtype):
    """Operands whose logits are multiples of 1/8 below 2^10: exact in fp32, in whatever order they are summed."""
    draw = lambda n: torch.randint(-1, 2, (n, k), generator=g, device=g.device)  # noqa: E731
    return draw(t).to(DT[dtype]), (draw(v) / 8).to(DT[dtype])


def _gen(dev, seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def _reference(hidden, weight, targets):
    z = hidden.double() @ weight.double().t().contiguous()
    lse = torch.logsumexp(z, 1)
    return z.gather(1, targets.long().clamp(0, weight.shape[0] - 1)[:, None])[:, 0] - lse, lse


def _check(got, want, extra=0.0):
    for x, y in zip(got, want):
        bound = 2.0**-24 * (120 + 4 * y.abs() + 4 * want[1].abs()) + extra
        worst = ((x.double() - y).abs() / bound).max().item()
        assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("t", [1, 2, 15, 16, 17, 33, 64, 65, 128, 129, 255, 256, 257, 700])
@pytest.mark.parametrize("v,k", [(1, 64), (7, 128), (127, 192), (257, 64), (1003, 512), (4099, 320)])
def test_sizes(gpu, t, v, k, dtype):
    g = _gen(gpu, t)
    hidden, weight = _whole(g, t, v, k, dtype)
    targets = torch.randint(0, v, (t,), generator=g, device=gpu)
    targets[0], targets[-1] = v - 1, 0
    want = _reference(hidden, weight, targets)
    _check(token_logprobs(hidden, weight, targets), want)
    _check(token_logprobs(hidden, weight, targets.int()), want)


@pytest.mark.parametrize("t", [3, 40, 100, 300, 2100])
def test_the_model_s_sizes(gpu, t):
    """Hidden states and weights of ordinary values, logits of up to 12; many token tiles beside each other."""
    g = _gen(gpu, 2)
    k, v = 3584, 20011
    hidden = torch.randn((t, k), generator=g, device=gpu).half()
    weight = (torch.randn((v, k), generator=g, device=gpu) * (2.5 / math.sqrt(k))).half()
    targets = torch.randint(0, v, (t,), generator=g, device=gpu)
    size = (hidden.abs().float() @ weight.abs().float().t()).max().item()
    got = token_logprobs(hidden, weight, targets)
    want = _reference(hidden, weight, targets)
    _check(got, want, 2 * k * 2.0**-24 * size)
    # and as near as plain fp32 sums are: an error of that size grows with the square root of K
    assert max((x.double() - y).abs().max().item() for x, y in zip(got, want)) <= 2 * math.sqrt(k) * 2.0**-24 * size


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("t", [130, 160, 161, 319, 320, 321, 384, 385, 640, 641, 799])
def test_tiles_of_tokens(gpu, t, dtype):
    """Widths of the tiles of many tokens and their neighbours, each token its own target."""
    g = _gen(gpu, t)
    hidden, weight = _whole(g, t, 777, 128, dtype)
    targets = torch.arange(t, device=gpu) % 777
    _check(token_logprobs(hidden, weight, targets), _reference(hidden, weight, targets))


@pytest.mark.parametrize("t", [1, 50, 90, 300])
def test_likely_tokens_and_large_logits(gpu, t):
    """Logits of thousands, a target that has nearly all of the probability: z - lse must not lose it."""
    g = _gen(gpu, 3)
    hidden, weight = _whole(g, t, 900, 256, "fp16")
    weight = weight * 64                                 # multiples of 8 up to 2048
    targets = (hidden.double() @ weight.double().t()).argmax(1)
    want = _reference(hidden, weight, targets)
    got = token_logprobs(hidden, weight, targets)
    assert torch.isfinite(torch.stack(got)).all()
    _check(got, want)
    # next to 0 the result's own size counts, not lse's: the sum of the others' exponentials, 1e-6 of it
    near = want[0].abs() < 0.1
    assert ((got[0].double() - want[0])[near].abs() <= 2.0**-20).all()


@pytest.mark.parametrize("t", [9, 200])
def test_targets_outside_and_values_that_are_not_finite(gpu, t):
    g = _gen(gpu, 4)
    hidden, weight = _whole(g, t, 300, 128, "fp16")
    targets = torch.randint(0, 300, (t,), generator=g, device=gpu)
    want = _reference(hidden, weight, targets)
    targets[0], targets[1], targets[2], targets[3] = -1, 300, 2**40, -2**62
    got = token_logprobs(hidden, weight, targets)
    assert got[0][0] == 0 and got[0][3] == 0 and torch.isnan(got[0][1:3]).all()
    _check([x[4:] for x in got], [x[4:] for x in want])
    _check([got[1]], [want[1]] * 2)
    hidden[4] = math.nan
    got = token_logprobs(hidden, weight, targets)
    assert torch.isnan(got[0][4]) and torch.isnan(got[1][4])
    _check([x[5:] for x in got], [x[5:] for x in want])
    # a logit of infinity: that of the one weight row that is (only its column of the product)
    hidden, weight = _whole(g, t, 300, 128, "fp16")
    hidden[:, 0] = 1
    weight[17, 0] = math.inf
    targets = torch.full((t,), 3, device=gpu)
    got = token_logprobs(hidden, weight, targets)
    assert (got[1] == math.inf).all() and (got[0] == -math.inf).all()
    weight[17, 0] = -math.inf                            # one token less
    got = token_logprobs(hidden, weight, targets)
    _check(got, _reference(hidden, weight[torch.arange(300, device=gpu) != 17], targets))


def test_strides_streams_and_repeats(gpu):
    g = _gen(gpu, 5)
    for t in (3, 60, 120, 400):
        hidden, weight = _whole(g, t, 1000, 192, "bf16")
        targets = torch.randint(0, 1000, (t,), generator=g, device=gpu)
        want = token_logprobs(hidden, weight, targets)
        wide = torch.zeros((t, 1024), dtype=hidden.dtype, device=gpu)
        wide[:, 64:256] = hidden
        odd = torch.zeros(weight.numel() + 1, dtype=weight.dtype, device=gpu)
        odd[1:] = weight.reshape(-1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = [token_logprobs(wide[:, 64:256], odd[1:].view(weight.shape), targets) for _ in range(3)]
        here = [token_logprobs(hidden, weight, targets) for _ in range(3)]
        torch.cuda.synchronize()
        for got in other + here:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_in_a_graph(gpu):
    g = _gen(gpu, 6)
    for t in (4, 300):
        hidden, weight = _whole(g, t, 777, 128, "fp16")
        targets = torch.randint(0, 777, (t,), generator=g, device=gpu)
        token_logprobs(hidden, weight, targets)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = token_logprobs(hidden, weight, targets)
        torch.cuda.current_stream().wait_stream(side)
        for k in range(4):
            hidden.copy_(_whole(_gen(gpu, 60 + k), t, 1, 128, "fp16")[0])
            want = token_logprobs(hidden, weight, targets)
            out[0].zero_()
            out[1].zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), k
            _check(out, _reference(hidden, weight, targets))


@pytest.mark.parametrize("t", [2, 130])
def test_weights_past_32_bits(gpu, t):
    """A projection of 4.7 GB: the last rows are found."""
    g = _gen(gpu, 7)
    v, k = 1150011, 2048
    weight = torch.zeros((v, k), dtype=torch.float16, device=gpu)
    hidden = torch.randint(-1, 2, (t, k), generator=g, device=gpu).half()
    weight[-5:] = (torch.randint(-1, 2, (5, k), generator=g, device=gpu) / 8).half()
    targets = torch.arange(t, device=gpu) % 5 + (v - 5)
    z = hidden.double() @ weight[-5:].double().t().contiguous()
    rest = torch.full((t, 1), math.log(v - 5), dtype=torch.float64, device=gpu)
    lse = torch.logsumexp(torch.cat((z, rest), 1), 1)
    _check(token_logprobs(hidden, weight, targets), (z.gather(1, (targets - (v - 5))[:, None])[:, 0] - lse, lse))


def test_no_tokens_and_refusals(gpu):
    g = _gen(gpu, 8)
    hidden, weight = _whole(g, 3, 50, 64, "fp16")
    targets = torch.zeros(3, dtype=torch.int64, device=gpu)
    assert [x.shape for x in token_logprobs(hidden[:0], weight, targets[:0])] == [(0,), (0,)]
    for a in ((hidden.float(), weight.float(), targets), (hidden, weight.bfloat16(), targets), (hidden[0], weight, targets),
              (hidden, weight[:, :32], targets), (hidden[:, :32], weight[:, :32], targets), (hidden, weight[:0], targets),
              (hidden.cpu(), weight, targets), (hidden, weight.cpu(), targets), (hidden, weight, targets.cpu()),
              (hidden, weight, targets[:2]), (hidden, weight, targets.float()), (hidden, weight, targets[:, None])):
        with pytest.raises(ValueError):
            token_logprobs(*a)
    assert _native.lib().awq_serve_logprobs_workspace(0, 5) == 0

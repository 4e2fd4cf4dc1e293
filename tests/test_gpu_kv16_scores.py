"""Scores of the 16-bit cache's attention (``kernels/kv16.py``) at the ends of fp32, against 64 bits."""
import kv16_oracle as O
import pytest
import torch
from test_gpu_kv16 import _batch, _call, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("tokens", [300, 3000])
@pytest.mark.parametrize("scale", [768.0, 1e30, 3e38])
def test_distances_under_large_scales(gpu, rows, tokens, scale):
    """bf16 queries of 2^125, brought down by 2^118, under scales whose product with that is near fp32's largest number
    or past it: keys of zero have a score of zero, and the distances alone weigh the tokens.  With keys of 2^-126 a
    scale of 768 gives scores 384 apart, all of them inside fp32."""
    g = _gen(gpu, 21)
    q, cache, tables, lens, starts = _batch(g, [(tokens, rows), (64, 1)], nh=2, kvh=1, hd=128, page=64, dtype="bf16")
    q = torch.where(q < 0, -(2.0**125), 2.0**125).to(torch.bfloat16)
    cache.k.zero_()
    slopes = torch.tensor([0.5, 0.03], device=gpu)
    args = (q, cache, tables, lens, starts)
    O.check(_call(*args, scale=scale, slopes=slopes), *O.attention(q, cache.data, *args[2:], scale=scale, slopes=slopes), "zeros")
    if scale == 768.0:
        cache.k.copy_(torch.randint(-1, 2, cache.k.shape, generator=g, device=gpu) * 2.0**-126)
        O.check(_call(*args, scale=scale, slopes=slopes), *O.attention(q, cache.data, *args[2:], scale=scale, slopes=slopes), "small")


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("tokens", [300, 3000])
@pytest.mark.parametrize("softcap", [None, 30.0])
def test_large_keys_under_large_scales(gpu, rows, tokens, softcap):
    """Queries of 2^125 and keys of 2^40 under 1e30: products sum inside fp32 all the same.  Plain, the largest score has all of the
    weight; capped, every positive score is the cap and all other tokens weigh e^-60 at most."""
    g = _gen(gpu, 22)
    q, cache, tables, lens, starts = _batch(g, [(tokens, rows), (64, 1)], nh=2, kvh=1, hd=128, page=64, dtype="bf16")
    q = (q.float() * 2.0**125).to(torch.bfloat16)
    cache.k.copy_((cache.k.float() * 2.0**40).to(torch.bfloat16))
    args = (q, cache, tables, lens, starts)
    out = _call(*args, scale=1e30, softcap=softcap)
    y, _ = O.attention(q, cache.data, *args[2:], scale=1e30, softcap=softcap)
    assert torch.isfinite(out).all()
    # a rounding of the probabilities (equal ones), of the result, and of sums of up to 3000 terms
    assert (out.double().view(y.shape) - y).abs().max() <= 3 * 2.0**-9 * cache.v.abs().max()

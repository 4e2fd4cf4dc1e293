"""Chunks beside many single tokens over the 16-bit cache (``kernels/kv16.py``): both kernels have a share and the chunk is split,
against 64 bits."""
import kv16_cuts
import kv16_oracle as O
import pytest
from test_gpu_kv16 import _batch, _call, _features, _gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cuts(tmp_path_factory):
    return kv16_cuts.build(tmp_path_factory.mktemp("cuts16"))


@pytest.mark.parametrize("features", ["", "cap slopes window prefix first"])
@pytest.mark.parametrize("nh,kvh,hd,page,dtype,requests", [
    (28, 4, 128, 64, "fp16", [(200 + 7 * i, 1) for i in range(64)] + [(6000, 300)]),
    (14, 2, 64, 16, "bf16", [(7000, 150)] + [(1 + 13 * i % 500, 1) for i in range(130)] + [(3000, 77)]),
    (8, 1, 128, 32, "fp16", [(300, i % 3) for i in range(70)] + [(4000, 40)] + [(90, 2)] * 5)])
def test_a_chunk_beside_many_tokens(gpu, cuts, nh, kvh, hd, page, dtype, requests, features):
    c = cuts(requests, nh // kvh, kvh, page=page).check()
    assert c.decode_items and c.tile_items and c.tile_splits > 1, c
    g = _gen(gpu, 31)
    args = _batch(g, requests, nh=nh, kvh=kvh, hd=hd, page=page, dtype=dtype, gain=4.0 if "cap" in features else 1.0)
    kw = _features(g, features.split(), nh, args[3], args[4])
    O.check(_call(*args, **kw), *O.attention(args[0], args[1].data, *args[2:], **kw))

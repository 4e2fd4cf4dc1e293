"""How the attention of the 16-bit cache cuts its work, as its kernels do it, on the host (``attention16_cuts.cpp``)."""
import random

import kv16_cuts
import kv16_plans
import pytest


@pytest.fixture(scope="session")
def cuts(tmp_path_factory):
    return kv16_cuts.build(tmp_path_factory.mktemp("cuts16"))


@pytest.mark.parametrize("window", [0, 1, 100, 4096, 2**31 - 2])
@pytest.mark.parametrize("requests,group,kvh", [
    ([(2**30, 1)], 7, 4), ([(2**30, 4096)], 7, 4), ([(2**31 - 1, 1)], 8, 8), ([(2**30 - 1, 1)] * 4096, 1, 768),
    ([(2**29 + 65, 70), (1, 1), (2**29 + 1, 9), (3, 5)], 64, 1), ([(1, 1)], 1, 1), ([(0, 0), (0, 3)], 4, 2),
    ([(2**30 - 1, 40)] * 70, 7, 4), ([(2**30 - 1, 1)] * 200 + [(2**30 - 1, 300)], 7, 4)])
def test_the_longest(cuts, requests, group, kvh, window):
    cuts(requests, group, kvh, window=window, page=256, width=min(2**22, -(-max(n for n, _ in requests) // 256) or 1)).check()


def test_many_shapes(cuts):
    rng = random.Random(3)
    for _ in range(1500):
        longest, most = rng.choice([1, 100, 5000, 200000]), rng.choice([1, 4, 60, 700, 3000])
        requests = [(rng.choice([0, rng.randint(1, longest)]), rng.choice([0, 1, 1, rng.randint(1, most)]))
                    for _ in range(rng.choice([1, 1, 2, 5, 64, 65, 300]))]
        if rng.random() < 0.3:                          # prompts
            requests = [(m, m) for _, m in requests]
        kw = {"total": max(0, sum(m for _, m in requests) + rng.choice([0, 0, 9, -3])), "page": rng.choice([16, 64, 256]),
              "window": rng.choice([0, rng.randint(1, longest + 5)])}
        if rng.random() < 0.2:
            kw["max_query"] = rng.randint(1, most)
        if rng.random() < 0.2:
            kw["width"] = rng.randint(1, 20)
        cuts(requests, rng.choice([1, 4, 7, 8, 64]), rng.choice([1, 4, 8, 40]), **kw).check()


@pytest.mark.parametrize("steps", [1, 2, 3, 15, 16, 17, 63, 64, 65, 100, 1000, 4095])
def test_one_request_of_every_row_count(cuts, steps):
    """Lengths around a whole number of steps, chunks from few rows to many, one request."""
    for tail in (1, 37, 64):
        for rows in (19, 40, 150, 300, 700):
            n = 64 * (steps - 1) + tail
            if rows <= n:
                cuts([(n, rows)], 7, 4).check()
                cuts([(n, n)], 7, 4).check()


@pytest.mark.parametrize("decodes", [0, 1, 8, 32, 64, 200])
def test_a_chunk_beside_single_tokens_keeps_its_split(cuts, decodes):
    """300 rows behind 32768 tokens are 17 blocks of a kv head: whole, each would walk over all of the tokens by itself."""
    for single in (1, 2000):
        c = cuts([(single + 7 * i, 1) for i in range(decodes)] + [(32768, 300)], 7, 4).check()
        assert c.tile_sums and c.parts == 1 and c.tile_splits >= 4 and c.tile_longest <= 128, c
    # in front of the chunk, and several chunks
    c = cuts([(32768, 300)] + [(500, 1)] * decodes + [(20000, 150)], 7, 4).check()
    assert c.tile_sums and c.tile_splits >= 2, c


@pytest.mark.parametrize("name", kv16_plans.PLANS)
def test_the_batches_of_the_long_plans(cuts, name):
    """What ``kv16_plans`` says of each of its batches."""
    nh, kvh, _, page, requests, want = kv16_plans.PLANS[name]
    c = cuts(requests, nh // kvh, kvh, page=page).check()
    assert {k: getattr(c, k) for k in want} == want, c
    if name.startswith("split"):
        assert c.tile_splits > 1 and c.tile_longest * 64 > 64 * page, c

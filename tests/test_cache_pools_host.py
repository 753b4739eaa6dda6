"""The page operations refuse pools that share memory, checked against the
addresses themselves."""
import random

import pytest
import torch

import ops_b200
from ops_b200.cache import _pools_meet
from test_cache_host import CALLS, GOOD


def test_against_addresses():
    r, seen = random.Random(3), {True: 0, False: 0}
    for _ in range(6000):
        pages = r.randint(1, 5)
        stride = r.randint(1, 12)
        pools = []
        for _ in range(r.randint(1, 4)):
            size = r.randint(0, stride)
            pools.append((r.randint(1, 60), stride if r.random() < 0.7 else size or 1, size))
        sets = [{b + p * s + i for p in range(pages) for i in range(n)} for b, s, n in pools]
        want = sum(map(len, sets)) > len(set().union(*sets))
        if any(s < n for _, s, n in pools):
            continue                               # pages that overlap are refused before
        got = _pools_meet([x for p in pools for x in p], pages)
        # pools of other strides inside one another are refused even where their pages miss each other
        assert got == want or (got and len({s for _, s, n in pools if n}) > 1), (pages, pools)
        seen[want] += 1
    assert min(seen.values()) > 500


BUF = torch.zeros(20, 8, 2)
HALVES = torch.zeros(6, 2, 8, 2)


@pytest.mark.parametrize("op", ["fork", "accept", "compact", "copy"])
@pytest.mark.parametrize("pools,msg", [
    ([BUF[:6], BUF[1:7]], "share memory"),                     # shifted by a page
    ([BUF[1:7], BUF[8:14], BUF[:6]], "share memory"),
    ([HALVES[:, 0], HALVES.view(12, 8, 2)[2:8]], "share memory"),
    ([BUF[:6], BUF[6:12], BUF[12:18]], "CUDA"), ([HALVES[:, 0], HALVES[:, 1]], "CUDA"), ([HALVES[:, 1], HALVES[:, 0]], "CUDA"),
    ([HALVES[:, 1], torch.zeros(6, 8, 5), HALVES[:, 0], torch.zeros(6, 8, 0)], "CUDA"),
])
def test_refusals(op, pools, msg):
    with pytest.raises(ValueError, match=msg):
        CALLS[op]({**GOOD, "pools": pools})

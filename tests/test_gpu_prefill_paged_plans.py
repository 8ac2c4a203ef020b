"""Prefill over a paged cache: what lies past the last key that a tile of queries sees."""
import math

import pytest
import torch

from inkling_fa4 import inkling_fa4_rel_attention_paged
from paged_cases import F8, Case

pytestmark = pytest.mark.gpu


def run(c, dev, max_q=None, max_k=None):
    print("paged plans:", c.told(), flush=True)
    out, lse = inkling_fa4_rel_attention_paged(*c.on(dev), max_q or c.max_q, max_k or c.max_k,
                                               c.extent, causal=c.causal, **c.settings())
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


# a tile of 128 rows ends inside a tile of 64 keys; packed heads; cut into chunks; a window
@pytest.mark.parametrize("news,lens,window", [([140], [150], -1), ([140, 300], [150, 333], -1),
                                              ([300], [5010], -1), ([300], [777], 100),
                                              ([200] * 5, [210] * 5, -1)])
@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("rel", ["token", "table"])
def test_keys_that_no_query_of_a_tile_sees(cuda, news, lens, window, kv, rel):
    """Later tokens' keys and values may be infinite or NaN: the tiles before them do not notice."""
    c = Case(news, lens, window=window, kv=kv, rel=rel, seed=36)
    clean = run(c, cuda)
    for b, (n, lk) in enumerate(zip(news, lens)):
        past = lk - n + 128  # the first key past the first tile's last query
        j = torch.arange(past, lk)
        at = c.table[b, j // c.block].long()
        c.kc[at, j % c.block] = torch.tensor(math.nan).to(c.kc.dtype)
        c.vc[at, j % c.block] = torch.tensor(math.nan if kv else math.inf).to(c.vc.dtype)
    out, lse = run(c, cuda)
    start = 0
    for n in news:
        assert torch.equal(out[start:start + 128], clean[0][start:start + 128])
        assert torch.equal(lse[:, start:start + 128], clean[1][:, start:start + 128])
        start += n

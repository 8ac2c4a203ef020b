"""Windows and lengths past 31 bits: a window so wide is none, a length so long is refused."""
import pytest
import torch

from inkling_fa4 import (inkling_fa4_rel_attention_decode_paged, inkling_fa4_rel_attention_paged,
                         inkling_fa4_rel_attention_sparse_paged)
from paged_cases import Case

pytestmark = pytest.mark.gpu


def call(c, args, op, max_q=None, max_k=None, extent=None, **kw):
    kw = dict(c.settings(), **kw)
    if op is inkling_fa4_rel_attention_sparse_paged:
        args = args + [torch.arange(40, dtype=torch.int32, device=args[0].device).expand(
            args[0].shape[0], c.hkv, 40).contiguous()]
    if op is inkling_fa4_rel_attention_decode_paged:
        kw["bottom_right"] = True
    return op(*args, c.max_q if max_q is None else max_q, c.max_k if max_k is None else max_k,
              c.extent if extent is None else extent, **kw)


@pytest.mark.parametrize("op", [inkling_fa4_rel_attention_paged, inkling_fa4_rel_attention_sparse_paged,
                                inkling_fa4_rel_attention_decode_paged])
def test_wide_windows_and_lengths(cuda, op):
    c = Case([1, 1] if op is inkling_fa4_rel_attention_decode_paged else [30, 4], [400, 500], seed=2)
    args = c.on(cuda)
    want = call(c, args, op)
    for wide in (2 ** 31, 2 ** 32, 2 ** 32 + 7, 2 ** 62):
        got = call(c, args, op, window_size=(wide, 0))
        torch.testing.assert_close(got[0].float(), want[0].float(), atol=1e-3, rtol=1e-2)
        torch.testing.assert_close(got[1], want[1], atol=1e-5, rtol=0)
    for kw in (dict(max_q=2 ** 32 + 30), dict(max_k=2 ** 32 + 500), dict(extent=2 ** 32 + 128),
               dict(extent=2 ** 32), dict(max_k=-1), dict(max_q=-(2 ** 32) + 30)):
        with pytest.raises((RuntimeError, ValueError)):
            call(c, args, op, **kw)
    torch.cuda.synchronize()

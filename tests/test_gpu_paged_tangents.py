"""The attentions over a paged cache have no derivative: a tangent is refused, it does not vanish, and
outputs never require a gradient."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from inkling_fa4 import inkling_fa4_rel_attention_paged, inkling_fa4_rel_attention_sparse_paged
from paged_cases import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("which", range(4))
def test_tangents_and_gradients(cuda, sparse, which):
    c = Case([3, 4], [40, 50], seed=1)
    args = c.on(cuda)
    lists = torch.arange(4, dtype=torch.int32, device=cuda).expand(7, c.hkv, 4).contiguous()
    op = inkling_fa4_rel_attention_sparse_paged if sparse else inkling_fa4_rel_attention_paged

    def call(*a):
        return op(*a, *([lists] if sparse else []), c.max_q, c.max_k, c.extent, **c.settings())

    want = call(*args)
    with fwad.dual_level():
        dual = list(args)
        dual[which] = fwad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(*dual)
    args[which] = args[which].clone().requires_grad_()
    got = call(*args)
    assert not got[0].requires_grad and not got[1].requires_grad
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

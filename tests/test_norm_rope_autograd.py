"""Head norm and paged append under autograd (CPU): the binding's autograd kernels above stand-ins
for the GPU's, which are linear in q and k, or fill the caches."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from inkling_fa4 import inkling_fa4_kv_append_paged, inkling_fa4_qk_norm_rope
from inkling_fa4._native import ops


@pytest.fixture
def stand_ins():
    ops()
    lib = torch.library.Library("inkling_fa4", "IMPL")

    def append(k, v, k_cache, v_cache, cu, used, table, q, *rest):
        with torch.no_grad():  # as the kernel: writes that autograd does not see
            for cache in (k_cache, v_cache):
                cache.data.fill_(7.0)
        return 2 * q if q is not None else k.new_empty(0)
    lib.impl("qk_norm_rope", lambda q, k, *rest: (2 * q, 3 * k), "CPU")
    lib.impl("kv_append_paged", append, "CPU")
    yield
    lib._destroy()


def _heads():
    g = torch.Generator().manual_seed(1)
    return torch.randn(3, 2, 64, generator=g), torch.randn(3, 1, 64, generator=g)


@pytest.mark.parametrize("which", range(4))
def test_forward_mode_is_refused(stand_ins, which):
    """A tangent of q, k or a weight is refused; it does not vanish."""
    x = list(_heads()) + [torch.ones(64), torch.ones(64)]
    with fwad.dual_level():
        dual = [fwad.make_dual(t, torch.ones_like(t)) if i == which else t for i, t in enumerate(x)]
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(NotImplementedError, match="forward"):
                inkling_fa4_qk_norm_rope(*dual)

    def f(t):
        return inkling_fa4_qk_norm_rope(*(t if i == which else y for i, y in enumerate(x)))
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(f, (x[which],), (torch.ones_like(x[which]),))
    for a, b in zip(inkling_fa4_qk_norm_rope(*x), (2 * x[0], 3 * x[1])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("which", ["q", "k", "v", "k_weight"])
def test_forward_mode_of_the_append_is_refused(stand_ins, which):
    q, k = _heads()
    cache, ints = torch.zeros(4, 16, 1, 64), torch.zeros(2, dtype=torch.int32)
    named = dict(q=q, k=k, v=k.clone(), k_weight=torch.ones(64))
    with fwad.dual_level():
        named[which] = fwad.make_dual(named[which], torch.ones_like(named[which]))
        with pytest.raises(NotImplementedError, match="forward"):
            inkling_fa4_kv_append_paged(**named, k_cache=cache, v_cache=cache.clone(),
                                        cu_seqlens_q=ints, seqused_k=ints[:1], block_table=ints[None])

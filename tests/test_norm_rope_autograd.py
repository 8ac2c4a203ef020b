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


def _append_call(q, k, kc, vc, **kw):
    ints = torch.zeros(2, dtype=torch.int32)
    return inkling_fa4_kv_append_paged(k, k.clone(), kc, vc, ints, ints[:1], ints[None], q=q, **kw)


def test_a_graph_that_saved_the_cache_notices_the_append(stand_ins):
    """The caches change in place, as autograd sees it: their versions go up, and a backward pass
    that needs what they held raises."""
    q, k = _heads()
    for mode in (torch.enable_grad, torch.no_grad, torch.inference_mode):
        kc, vc = torch.ones(4, 16, 1, 64), torch.ones(4, 16, 1, 64)
        x = torch.ones_like(kc, requires_grad=True)
        y = (x * kc).sum() + (x * vc).sum()
        before = kc._version, vc._version
        with mode():
            _append_call(q, k, kc, vc)
        assert kc._version > before[0] and vc._version > before[1] and kc.eq(7).all()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    both = torch.ones(2, 4, 16, 1, 64)  # views of one pool share its version
    before = both._version
    _append_call(q, k, both[0], both[1])
    assert both._version > before


def test_caches_that_require_a_gradient_are_refused(stand_ins):
    q, k = _heads()
    for leaf in (True, False):
        for which in (0, 1):
            caches = [torch.ones(4, 16, 1, 64), torch.ones(4, 16, 1, 64)]
            caches[which].requires_grad_()
            if not leaf:
                caches[which] = 2 * caches[which]
            held = caches[which].detach().clone()
            with pytest.raises(RuntimeError, match="require"):
                _append_call(q, k, *caches)
            assert torch.equal(caches[which].detach(), held)
            with torch.no_grad():  # as any in-place write
                _append_call(q, k, *caches)
            assert caches[which].detach().eq(7).all()


def test_caches_made_in_inference_mode(stand_ins):
    """They have no version to go up."""
    q, k = _heads()
    with torch.inference_mode():
        kc, vc = torch.ones(4, 16, 1, 64), torch.ones(4, 16, 1, 64)
        out = _append_call(q, k, kc, vc)
    assert torch.equal(out, 2 * q) and kc.eq(7).all()
    assert torch.equal(_append_call(q, k, kc, vc), 2 * q)

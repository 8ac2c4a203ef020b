"""Decode behind a shared prefix under plans that the shorter calls of test_gpu_decode_shared.py do
not get (PLANS of test_shared_plan.py, which pins what they are), against the definition in fp64
with the same bounds."""
import pytest
import torch

from test_gpu_decode_shared import F8, Case
from test_shared_plan import PLANS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", [None, F8])
@pytest.mark.parametrize("name", list(PLANS))
def test_plans(cuda, name, kv):
    lens, prefix, hq, hkv, window, extent = PLANS[name]
    c = Case(lens, prefix, hq, hkv, 64, block=64, kv=kv, window=window, extent=extent, seed=len(lens))
    c.check(c.run(cuda))


@pytest.mark.parametrize("window", [-1, 300])
def test_a_length_past_the_table_counts_as_the_table(cuda, window):
    """seqused_k past the table's columns: the result of as many keys as the table holds, bias
    distances and window counted from there; a negative one is an empty sequence."""
    c = Case([704, 704, 640], 640, extent=200, window=window, seed=10)
    want = c.run(cuda)
    c.check(want)
    c.used = torch.tensor([10 ** 6, 2 ** 31 - 1, -5], dtype=torch.int32)
    c.lens = [704, 704, 0]
    got = c.run(cuda)
    c.check(got)
    assert torch.equal(got[0][:2], want[0][:2]) and torch.equal(got[1][:, :2], want[1][:, :2])

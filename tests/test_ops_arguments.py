"""CPU tests of verbo_b200/ops.py: numbers that the C ABI's ints do not hold are
refused, not taken modulo 2^32."""
from __future__ import annotations

import copy
import pickle

import pytest

import verbo_b200 as vb

torch = pytest.importorskip("torch")

WIDE = [2**31, 2**32 + 32, -2**31 - 1, 2**63]


@pytest.mark.parametrize("group", WIDE)
def test_group(group):
    q, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.float16)
    with pytest.raises(vb.VerboCudaError, match="group must be"):
        vb.Q4Linear(q, s, group=group, device="cuda:0")


@pytest.mark.parametrize("last", WIDE)
def test_window(last):
    with pytest.raises(vb.VerboCudaError, match="last"):
        vb.Penalties(1.1, last=last)
    assert vb.Penalties(1.1, last=2**31 - 1).last == 2**31 - 1
    assert vb.Penalties(1.1, last=-2**31).last == -2**31


@pytest.mark.parametrize("top", [33, -1, *WIDE])
def test_top(top):
    """Before the results are allocated."""
    with pytest.raises(vb.VerboCudaError, match="top"):
        vb.token_logprobs(torch.zeros(2, 8), top=top)


@pytest.mark.parametrize("shape", [(2**31, 1), (2**32 + 2, 1), (1, 2**32 + 8)])
def test_rows_and_columns(shape):
    x = torch.zeros(1, 1).expand(*shape)
    with pytest.raises(vb.VerboCudaError, match="2147483647"):
        vb.process_logits(x)
    with pytest.raises(vb.VerboCudaError, match="2147483647"):
        vb.token_logprobs(x, top=1)


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, pickle.dumps], ids=["copy", "deepcopy", "pickle"])
def test_a_layer_is_not_copied(how):
    """A second object with the handle would free it a second time."""
    layer = object.__new__(vb.Q4Linear)
    layer._h = None
    with pytest.raises(TypeError, match="Q4Linear"):
        how(layer)

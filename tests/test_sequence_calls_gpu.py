"""Calls of the sequence operators that the other tests do not make: operands from the host, lazily negated, written in place; arguments of the C-ABI that
the Python entry points never hand over; waits between workgroups that fail."""
import ctypes as C
import math
import os
import sys

import numpy as np
import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, REPO)
from oracle import sequence_oracle as so  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dc():
    import dcarl_amd
    dcarl_amd.require_gpu()
    return dcarl_amd


def test_adjust_takes_histories_from_the_host(dc):
    s = torch.randn(3, 50, device="cuda")
    taken, off = [4, 4, 9, -1, 49], [0, 2, 2, 5]
    want = dc.candidates.adjust(s, torch.tensor(taken, device="cuda"), torch.tensor(off, device="cuda"), presence=0.5, frequency=0.25, repetition=1.5)
    assert torch.equal(dc.candidates.adjust(s, taken, off, presence=0.5, frequency=0.25, repetition=1.5, validate=True), want)
    assert torch.equal(dc.candidates.adjust(s, np.array(taken, dtype=np.int32), torch.tensor(off, device="cuda"), presence=0.5, frequency=0.25, repetition=1.5), want)
    changed = (want != s).nonzero().tolist()
    assert changed == [[0, 4], [2, 9], [2, 49]]


def test_adjust_in_place_is_seen_by_autograd(dc):
    p = torch.zeros(3, 40, device="cuda", requires_grad=True).exp()
    dc.candidates.adjust(p.detach(), bias=torch.ones(40, device="cuda"), out=p.detach())
    assert bool((p.detach() == 2).all())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        p.sum().backward()


def test_lazily_negated_operands(dc):
    z = torch.randn(40, 1, dtype=torch.complex64, device="cuda")
    x, off = z.conj().imag, [0, 11, 40]
    assert x.is_neg()
    want = dc.episodes.gated_recurrence(-z.imag, 0.5, off)
    assert torch.equal(dc.episodes.gated_recurrence(x, 0.5, off), want) and torch.equal(dc.episodes.gated_recurrence(x[:, 0], 0.5, off), want[:, 0])
    assert torch.equal(dc.tables.lookup(x, [3, 9, -1]), torch.cat([-z.imag[[3, 9]], torch.zeros(1, 1, device="cuda")]))
    assert torch.equal(dc.candidates.adjust(x), -z.imag)

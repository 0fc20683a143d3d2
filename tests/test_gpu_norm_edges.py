"""norm.block_norm and norm.rms_norm at the edges of what they take, next to the cases of tests/test_gpu_norm.py."""
import math

import pytest
import torch

from cinnamon_amd import _lib
from tests.test_gpu_norm import CASES, EPS, NAMES, call, check, definition, inputs


@pytest.mark.gpu
@pytest.mark.parametrize("gate", ["none", "channel", "row", "element"])
@pytest.mark.parametrize("shape", [(0, 128), (3, 0, 70)])
def test_no_rows_with_every_gate(dev, shape, gate):
    s, value, gn, gx = inputs(dev, shape, "bf16", "fp32", "fp32", True, gate, "channel")
    leaves = {k: t.clone().requires_grad_() for k, t in s.items() if t is not None}
    with torch.no_grad():
        n, x = call(s, value)
    assert n.shape == x.shape == shape and n.dtype == torch.bfloat16 and x.dtype == torch.float32
    n, x = call({**s, **leaves}, value)
    grads = dict(zip(leaves, torch.autograd.grad([n, x], list(leaves.values()), [gn, gx])))
    assert all(g.shape == s[k].shape and g.dtype == s[k].dtype for k, g in grads.items())
    assert all((grads[k] == 0).all() for k in NAMES[2:] if k in grads)


def test_c_entry_takes_no_rows_without_a_gate_pointer():
    lib = _lib.load()
    scale = (None, 0, 0, 1.0)
    for rows, kind, ok in ((0, 2, True), (0, 3, True), (0, 1, False), (4, 2, False), (4, 3, False)):
        args = (None, 0, 64, None, 0, 64, rows, 64, None, 0, None, 0, None, 0, kind, 64, *scale)
        want = 0 if ok else _lib.CIN_ERR_ARG
        assert lib.cin_block_norm(*args, EPS, None, None, None, None) == want, (rows, kind)
        assert lib.cin_block_norm_backward(*args, None, None, 0, None, 0, *(None,) * 6, None, 0, None) == want, (rows, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 128), (1, 1, 1100), (128,)])
def test_one_row_with_an_expanded_gate(dev, shape):
    """A gate that repeats one value has no stride, and of one row none that a copy would give it."""
    s, value, gn, gx = inputs(dev, shape, "bf16", "bf16", "fp32", False, "none", "one")
    gate = torch.full((), 0.625, device=dev).expand(*shape[:-1], 1)
    assert gate.stride()[-1] == 0
    results = []
    for g in (gate.clone(), gate.detach()):
        s["gate"] = g.requires_grad_()
        n, x = call(s, value)
        results.append((n, x, *torch.autograd.grad([n, x], [g], [gn, gx])))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert results[1][2].shape == gate.shape


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_gradients_within_their_own_sums(dev, case):
    """Each gradient by the roundings on its own way, beside the K of tests/test_gpu_norm.py (there a sum over a row is along
    16 + 6 + 16 of them; the forward's past 8192 channels is along 32 + 6 + 8, which K covers too):
      y, residual and a gate an element: none more;
      a gate a row: a sum over a row, 32 + 6 + 16;
      vectors: a workgroup's T / workgroups rows (at least 256 workgroups), a wave's three others, the
      partial rows in lines of 32 (at most 4096 / 32 a line) and the lines;
      a scale of one value: a thread's 16 channels of a row, the rest in 64 bits."""
    s, value, gn, gx = inputs(dev, *case)
    ref = definition(s, value, EPS, gn, gx)
    leaves = {k: t.clone().requires_grad_() for k, t in s.items() if t is not None}
    n, x = call({**s, **leaves}, value)
    outs, gs = ([n], [gn]) if x is None else ([n, x], [gn, gx])
    T = math.prod(case[0][:-1])
    vector = T / min(T, 256) + 3 + 4096 / 32 + 32
    more = {"y": 0, "residual": 0, "weight": vector, "post_weight": vector,
            "gate": {"channel": vector, "row": 32 + 6 + 16, "element": 0}.get(case[5]),
            "residual_scale": vector if case[6] == "channel" else 16}
    for k, g in zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gs)):
        check(g, ref[k], more[k])

"""The container of 8-bit blocks on the CPU: copies and pickles."""
import copy
import io
import pickle

import pytest
import torch


@pytest.fixture(scope="module")
def ops():
    from spn4cir_amd import ops as o
    return o


def saved(q):
    buf = io.BytesIO()
    torch.save({"w8": q}, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)["w8"]


@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda q: pickle.loads(pickle.dumps(q)), saved])
@pytest.mark.parametrize("rows", [0, 3])
def test_copies_of_blocks(ops, how, rows):
    """As the weights of a module that is copied or saved: the same bytes, checked like any other, and with copy() the same memory."""
    g = torch.Generator().manual_seed(0)
    q = ops.Fp8Blocks(torch.randint(0, 256, (rows, 256), dtype=torch.uint8, generator=g), torch.randint(0, 255, (rows, 4), dtype=torch.uint8, generator=g), 200)
    p = how(q)
    assert type(p) is ops.Fp8Blocks and p.K == 200 and p.rows == rows and torch.equal(p.data, q.data) and torch.equal(p.scale, q.scale)
    assert (p.data is q.data) == (how is copy.copy)
    with pytest.raises(AttributeError):
        p.K = 100

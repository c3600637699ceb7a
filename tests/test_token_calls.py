"""What the token operators' Python side owes to autograd, to tracing and to tensors that change hands (CPU: launches are
recorded instead of made), and calls of tests/test_tokens.py's operators that it leaves out (GPU)."""
import numpy as np
import pytest
import torch

DEV = 'cuda:0'


@pytest.fixture
def host(monkeypatch):
    """Rotary and KVCache over host tensors; the arguments of each launch are kept in the order of the calls."""
    from blast3r_amd import kv_cache, rotary
    calls = []

    def record(call, args, device):
        calls.append(type(args).from_buffer_copy(args))

    monkeypatch.setattr(torch.Tensor, 'is_cuda', True, raising=False)
    for m in (kv_cache, rotary):
        monkeypatch.setattr(m, 'launch', record)
    return calls


def _i32(x, device='cpu'):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)


# ---------------------------------------------------------------------------------- tensors written to

def test_tensors_written_to_count_as_changed(host):
    """Each tensor that a call writes to gets a new version, so that a backward that saved it raises."""
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.rotary import Rotary
    rot, pos = Rotary(64, device='cpu'), _i32([0, 1, 2])
    w = torch.ones(3, 2, 64, requires_grad=True)
    x, k = torch.randn(3, 2, 64), torch.randn(3, 1, 64)
    y = (w * x).sum()                                       # saves x
    with torch.no_grad():
        assert rot(pos, x, out=x) is x
    assert x._version == 1
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()
    rot(pos, x, k, out=(x, k))
    assert x._version == 2 and k._version == 1
    rot(pos, x, k)
    assert x._version == 2 and k._version == 1              # only read
    c = KVCache(2, 1, 64, device='cpu')
    q, pages, lens = torch.zeros(1, 2, 64, dtype=torch.bfloat16), _i32([[0, 1]]), _i32([5])
    held = (c.k, c.v, c.scales)
    before = [t._version for t in held]
    rows = torch.zeros(1, 1, 64)
    c.append(rows, rows, pages, lens)
    assert [t._version for t in held] == [v + 1 for v in before] and rows._version == 0
    out = torch.zeros_like(q)
    c.attend(q, pages, lens, out=out)
    c.read(pages, lens, None, 1)
    assert out._version == 1 and q._version == 0 and [t._version for t in held] == [v + 1 for v in before]
    with torch.inference_mode():                            # no versions there
        z = torch.zeros(3, 2, 64)
        rot(pos, z, out=z)
    with torch.no_grad():
        rot(pos, z, out=z)


def test_outputs_that_require_a_gradient_are_refused(host):
    from blast3r_amd.kv_cache import KVCache
    from blast3r_amd.rotary import Rotary
    rot, pos, x = Rotary(64, device='cpu'), _i32([0, 1, 2]), torch.randn(3, 2, 64)
    leaf = torch.zeros(3, 2, 64, requires_grad=True)
    with pytest.raises(ValueError, match='gradient'):
        rot(pos, x, out=leaf)
    with pytest.raises(ValueError, match='gradient'):
        rot(pos, x, x, out=(torch.zeros_like(x), leaf))
    c = KVCache(2, 1, 64, device='cpu')
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    out = torch.zeros_like(q).requires_grad_()
    with pytest.raises(RuntimeError, match='gradient'):
        c.attend(q, _i32([[0, 1]]), _i32([5]), out=out)
    assert not host
    with torch.no_grad():                                   # as torch's own operators take them
        rot(pos, x, out=leaf)
        c.attend(q, _i32([[0, 1]]), _i32([5]), out=out)
    assert len(host) == 2 and leaf._version == 1 and out._version == 1

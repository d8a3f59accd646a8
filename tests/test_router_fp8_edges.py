"""Corners of the router and FP8 operators that show without a GPU: what is refused, and before anything else."""
import pytest
import torch

import sm120fp4_b200 as pkg

fwd = torch.autograd.forward_ad


def test_forward_mode_is_refused():
    x, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: pkg.top_k_gate(dual, 2), lambda: pkg.top_k_gate(dual, 2, renormalize=False), lambda: pkg.balance_loss(dual, ids)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="GPU"):      # plain tensors get as far as ever
            pkg.top_k_gate(x, 2)


def test_the_host_extension_has_no_cxx_library_of_its_own():
    """Two C++ libraries in a process share some of their objects and not others: numbers written to a stream end it."""
    import sm120fp4_b200._lib as L
    host = L.host()
    assert host is not L.NO_HOST
    with open(host.__file__, "rb") as f:
        assert b"St7codecvtIDsc" not in f.read()      # (a part of the library that nothing here names)

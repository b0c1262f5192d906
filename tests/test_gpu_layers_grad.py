"""Gradients and tangents that the layers' calls do not have are refused, not lost
(MI355X)."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from rl_project_amd import qk_norm_rope, qk_norm_rope_backward, rotary_frequencies

pytestmark = pytest.mark.gpu


def test_frequencies_that_require_a_gradient():
    inv, _ = rotary_frequencies(16, device="cuda")
    q, pos = torch.randn(3, 2, 16, device="cuda"), torch.arange(3, device="cuda")
    want = qk_norm_rope(q, q, pos, inv)
    for dt in (torch.float64, torch.float32):
        leaf = inv.to(dt).requires_grad_(True)
        for x in (q, q.clone().requires_grad_(True)):
            with pytest.raises(RuntimeError, match="inv_freq"):
                qk_norm_rope(x, x, pos, leaf)
        with torch.no_grad():
            got = qk_norm_rope(q, q, pos, leaf)
        assert all(float((a - b).abs().max()) < 1e-5 for a, b in zip(got, want))
        assert torch.equal(qk_norm_rope(q, q, pos, leaf.detach())[0], got[0])
        qk_norm_rope_backward(q, q, q, q, pos, leaf)         # (the launches alone: records nothing)


def test_frequencies_with_a_tangent():
    inv, _ = rotary_frequencies(16, device="cuda")
    q, pos = torch.randn(3, 2, 16, device="cuda"), torch.arange(3, device="cuda")
    with fwAD.dual_level():
        dual = fwAD.make_dual(inv, torch.ones_like(inv))
        for call in (lambda: qk_norm_rope(q, q, pos, dual), lambda: qk_norm_rope_backward(q, q, q, q, pos, dual)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()

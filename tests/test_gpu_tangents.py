"""Forward-mode derivatives: none of the calls has one, and each says so rather than
return a result without its tangent (MI355X)."""

import pytest
import torch
import torch.autograd.forward_ad as fwad

from rl_project_amd import (layer_norm, layer_norm_backward, lm_head_logprobs, lm_head_logprobs_backward, score_tokens,
                            score_tokens_backward)

pytestmark = pytest.mark.gpu


def _calls():
    x = torch.randn(3, 70, device="cuda")
    tok = torch.zeros(3, dtype=torch.int64, device="cuda")
    w, b, dy = torch.ones(70, device="cuda"), torch.zeros(70, device="cuda"), torch.randn(3, 70, device="cuda")
    h = torch.randn(3, 64, device="cuda").bfloat16()
    head = torch.randn(90, 64, device="cuda").bfloat16()
    one = torch.ones(3, device="cuda")
    with torch.no_grad():
        _, stats = layer_norm(x, w, b, return_stats=True)
        _, saved = score_tokens(x, tok, return_saved=True)
        _, hsaved = lm_head_logprobs(h, head, tok, return_saved=True)
    return [
        (lambda x: score_tokens(x, tok, top_k=2), [x]),
        (lambda x, w, b: layer_norm(x, w, b), [x, w, b]),
        (lambda h, head: lm_head_logprobs(h, head, tok), [h, head]),
        (lambda x, saved, one: score_tokens_backward(x, tok, saved, one), [x, saved, one]),
        (lambda dy, x, w, stats: layer_norm_backward(dy, x, w, b, stats), [dy, x, w, stats]),
        (lambda h, head, hsaved, one: lm_head_logprobs_backward(h, head, tok, hsaved, one), [h, head, hsaved, one]),
    ]


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(grad):
    for call, args in _calls():
        for i in range(len(args)):
            with fwad.dual_level(), torch.set_grad_enabled(grad):
                call(*args)   # (no tangent: as ever)
                dual = list(args)
                dual[i] = fwad.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError):
                    call(*dual)


def test_tangents_of_an_upstream_gradient_are_refused():
    for call, args in _calls()[:3]:
        x = args[0].clone().requires_grad_()
        out = call(x, *args[1:])
        out = out if isinstance(out, torch.Tensor) else out.logprob
        with fwad.dual_level():
            up = fwad.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(out, x, up)


def test_tangents_beside_a_gradient_are_refused():
    for call, args in _calls()[:3]:
        for i in range(len(args)):
            leaves = [t.clone().requires_grad_() for t in args]
            with fwad.dual_level():
                leaves[i] = fwad.make_dual(leaves[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError):
                    call(*leaves)

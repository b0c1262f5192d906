"""The rank of a given token that is itself masked, or lower than any value the
kernel may put in the places past a row: with the entropy and without it, at
vocabularies that end inside a slice (MI355X).  Ranks are whole numbers and have
to be equal; the bounds of the other results are those of ``test_gpu_scores``."""

import math

import pytest
import torch

from rl_project_amd import score_tokens
from test_gpu_scores import DTYPES, H24, _near, _reference

pytestmark = pytest.mark.gpu

VOCABS = [5, 512, 1000, 4096, 16384, 16385, 32768, 50257, 128256]


def _case(V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = (2.5 * torch.randn(10, V, generator=g)).to(dtype)
    tok = torch.randint(0, V, (10,), generator=g)
    low = torch.finfo(dtype).min
    x[0, tok[0]] = -math.inf                                  # the row's only masked value
    x[1, tok[1]] = low                                        # the same with the type's lowest value
    gone = torch.rand(3, V, generator=g) < torch.tensor([[0.5], [0.9], [0.5]])
    x[2].masked_fill_(gone[0], -math.inf)[tok[2]] = -math.inf
    x[3].masked_fill_(gone[1], low)[tok[3]] = low
    x[4].masked_fill_(gone[2], low)[tok[4]] = -math.inf       # below the masks
    # below -1e30 (float16: its lowest values, a step apart)
    deep = {torch.float32: -1.5e30, torch.bfloat16: -1.5e30, torch.float16: -65472.0}[dtype]
    x[5, tok[5]] = deep
    x[6] = deep
    x[6, tok[6]] = 2 * deep if dtype != torch.float16 else low
    tok[7] = V - 1                                            # in the last slice, with the row's other masks in the first
    x[7, : min(V, 300)] = -math.inf
    x[7, -1] = -math.inf
    if V > 1:
        x[7, V - 2] = 1.0
    x[8] = -math.inf                                          # one value left, and it is not the token's
    tok[8] = 0
    x[8, V - 1] = 0.25
    x[9, tok[9]] = 30.0                                       # nothing above it
    return x, tok


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", VOCABS)
@pytest.mark.parametrize("entropy", [False, True])
def test_rank_of_a_masked_token(dtype, V, entropy):
    print(f"[rank] {dtype} V={V} entropy={entropy}", flush=True)
    x, tok = _case(V, dtype, V)
    ref = _reference(x, tok, 3)
    assert bool((ref["rank"] < V).all())
    xd, td = x.cuda(), tok.cuda()
    s = score_tokens(xd, td, top_k=3, entropy=entropy, lse=True, rank=True)
    assert s.rank.tolist() == ref["rank"].tolist()
    for name in ("lse", "logprob"):
        _near(getattr(s, name), ref[name], 66 * H24 + H24 * ref[name].abs().nan_to_num(0, 0, 0), name)
    if entropy:
        _near(s.entropy, ref["entropy"], ref["tol_h"], "entropy")
    assert torch.equal(s.top_ids.cpu(), ref["ids"])
    # what else is asked for does not depend on the rank
    t = score_tokens(xd, td, top_k=3, entropy=entropy, lse=True)
    for name in ("lse", "logprob", "top_logprobs") + (("entropy",) if entropy else ()):
        assert torch.equal(getattr(s, name), getattr(t, name)), name


def test_rank_beside_a_gradient_and_of_a_short_row():
    x = torch.zeros(2, 3, device="cuda")
    x[0, 1] = -math.inf
    tok = torch.tensor([1, 2], device="cuda")
    s = score_tokens(x.clone().requires_grad_(), tok, rank=True)
    assert s.rank.tolist() == [2, 0] and s.logprob.requires_grad
    assert float(s.logprob.detach()[0]) == -math.inf

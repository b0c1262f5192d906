"""lm_head_logprobs at sizes that take each tile of each product: the statistics
and the logits' gradient with 64, 128 and 256 rows, dweight with 64, 128 and 256
vocabulary rows, dhidden with its parts and without."""

import pytest
import torch

from rl_project_amd import lm_head_logprobs
from test_gpu_headlp import _inputs, _near, _ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,D,V", [
    (300, 1024, 2500),     # statistics 64, dweight 64
    (300, 1024, 8000),     # 64; 128
    (140, 256, 30000),     # 128; 128 (one tile of d)
    (100, 1024, 9001),     # 64; 256
    (129, 192, 33000),     # 256; 256 (one tile of d)
    (1100, 64, 8200),      # 256; 64
    (600, 320, 20000),     # 256; 256
])
def test_each_tile_against_float64(N, D, V):
    print(f"[tiles] {N}x{D}x{V}", flush=True)
    h, w, tok, ups = _inputs(N, D, V, N + D + V)
    ref = _ref(h, w, tok, ups)
    hd, wd = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    s = lm_head_logprobs(hd, wd, tok.cuda(), entropy=True, lse=True)
    for name in ("logprob", "entropy", "lse"):
        _near(getattr(s, name), ref[name], ref["t_" + name], name)
    a, b, c = (u.cuda() for u in ups)
    dh, dw = torch.autograd.grad((a * s.logprob + b * s.entropy + c * s.lse).sum(), (hd, wd))
    _near(dh, ref["dh"], ref["t_dh"], "dh")
    _near(dw, ref["dw"], ref["t_dw"], "dw")


def test_an_ignored_token_inside_the_vocabulary():
    h, w, tok, ups = _inputs(90, 128, 400, 3)
    tok = torch.where(tok < 0, torch.full_like(tok, 7), tok)
    tok[1] = 6
    ref = _ref(h, w, tok, ups, ignore=7)
    hd, wd = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    s = lm_head_logprobs(hd, wd, tok.cuda(), entropy=True, lse=True, ignore_index=7)
    _near(s.logprob, ref["logprob"], ref["t_logprob"], "logprob")
    assert bool((s.logprob.detach().cpu()[tok == 7] == 0).all())
    dh, dw = torch.autograd.grad((s.logprob, s.entropy, s.lse), (hd, wd), [u.cuda() for u in ups])
    _near(dh, ref["dh"], ref["t_dh"], "dh")
    _near(dw, ref["dw"], ref["t_dw"], "dw")


def test_rows_past_the_lists_of_a_vocabulary_row():
    """More rows of one token than are made good one by one, beside a row of
    another: the same bounds as without that."""
    h, w, tok, ups = _inputs(200, 128, 90, 5, scale=1.0)
    tok = torch.full_like(tok, 33)
    tok[150], tok[199] = 34, 89
    ref = _ref(h, w, tok, ups)
    hd, wd = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    s = lm_head_logprobs(hd, wd, tok.cuda(), entropy=True, lse=True)
    dh, dw = torch.autograd.grad((s.logprob, s.entropy, s.lse), (hd, wd), [u.cuda() for u in ups])
    _near(dh, ref["dh"], ref["t_dh"], "dh")
    _near(dw, ref["dw"], ref["t_dw"], "dw")

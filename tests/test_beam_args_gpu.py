"""What make_beam_select_args takes for scores in place: the score tensor's own words as
contiguous f32, one for each continuation, or nothing."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

GROUPS, WIDTH, VOCAB = 3, 4, 50


def _make(bh, dev, n_best=WIDTH, **kw):
    x = torch.randn((GROUPS * WIDTH, VOCAB), device=dev)
    wide = torch.zeros((GROUPS * WIDTH, 3), device=dev)
    score = wide.view(-1)[:GROUPS * WIDTH]
    return bh.make_beam_select_args(x, score, WIDTH, n_best,
                                    **{name: of(wide, score) for name, of in kw.items()})


def test_scores_in_place(bh, dev):
    for of in (lambda w, s: s, lambda w, s: s.view(GROUPS, WIDTH)):
        args = _make(bh, dev, score_out=of)
        assert args.score_out == args.score
        assert args.results[2].numel() == GROUPS * WIDTH


@pytest.mark.parametrize("what,of", [
    ("strided", lambda w, s: w[:, 0]),
    ("strided matrix", lambda w, s: w[:, 0].view(GROUPS, WIDTH)),
    ("integers", lambda w, s: s.view(torch.int32)),
    ("half as many", lambda w, s: s[:6]),
    ("more", lambda w, s: w.view(-1)),
    ("expanded", lambda w, s: s[:1].expand(GROUPS * WIDTH)),
])
def test_other_views_of_the_scores(bh, dev, what, of):
    with pytest.raises(ValueError, match="score_out"):
        _make(bh, dev, score_out=of)


def test_scores_in_place_where_n_best_is_not_width(bh, dev):
    with pytest.raises(ValueError, match="score_out may be score only where n_best is width"):
        _make(bh, dev, n_best=WIDTH + 1, score_out=lambda w, s: s)

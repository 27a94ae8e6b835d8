"""Ranges of chunks whose query heads are no whole fraction of a row tile: the heads of a token lie in two of them."""
import numpy as np
import pytest

import paged_oracle as po
from test_scoring_gpu import SCORES, ranges_of, run, slopes_of, status  # noqa: F401

pytestmark = pytest.mark.gpu


def first_and_last(tokens, group):
    """The tokens whose heads lie in two row tiles of 128 rows."""
    t = np.arange(tokens)
    return t * group // 128 != ((t + 1) * group - 1) // 128


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("kind", ["split", "documents", "prefix", "any"])
@pytest.mark.parametrize("d,mode,heads", [(128, 0, 2), (256, 3, 1)])
def test_ranges_of_any_group(cuda, status, group, kind, d, mode, heads):
    """Of the kind "split" every second token with heads in two row tiles sees everything, the others themselves alone: only they say how far a row tile walks."""
    rng = np.random.default_rng(10 * group + d + len(kind))
    lengths, tokens = [500, 333, 40], [260, 333, 1]
    pool = po.Pool(rng, lengths, d=d, heads=heads, page=32, mode=mode, qblock=32)
    if kind == "split":
        rows = []
        for n, length in zip(tokens, lengths):
            i = np.arange(length - n, length)
            far = first_and_last(n, group)
            far[np.flatnonzero(far)[::2]] = False
            rows.append(np.stack([np.where(far, 0, i), np.where(far, length, i + 1)], 1))
        ranges = np.concatenate(rows + [np.full((1, 2), 7)]).astype(np.int32)
    else:
        ranges = ranges_of(rng, kind, tokens, lengths, 1)
    scores = SCORES[group % 4]
    run(rng, pool, tokens, hq=heads * group, ranges=ranges, window=300 if group % 2 else 0, sinks=3 if group % 3 else 0, cap=scores.get("cap", 0.0),
        slopes=slopes_of(heads * group) if "slopes" in scores else None, word=status)


@pytest.mark.parametrize("group,tokens,base,start", [(3, 86, 43, 128), (5, 77, 13, 64), (7, 110, 55, 128)])
@pytest.mark.parametrize("d", [128, 256])
def test_a_document_that_begins_with_a_split_token(cuda, status, group, tokens, base, start, d):
    """The last token of a row tile, whose heads go on in the next one, is at the first position of a tile of the cache, and a document begins there."""
    rng = np.random.default_rng(group)
    token = start - base
    assert first_and_last(tokens, group)[token] and start % 64 == 0
    pool = po.Pool(rng, [base + tokens], d=d, heads=2, page=16, mode=0, qblock=32)
    i = np.arange(base, base + tokens)
    ranges = np.stack([np.where(i < start, 0, start), i + 1], 1).astype(np.int32)
    out, lse = run(rng, pool, [tokens], hq=2 * group, ranges=ranges, pad_rows=0, word=status)
    assert not bool(lse[token].isinf().any())
    ranges = np.stack([np.zeros(tokens, int), i + 1], 1).astype(np.int32)
    run(rng, pool, [tokens], hq=2 * group, ranges=ranges, pad_rows=0, word=status)

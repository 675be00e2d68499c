"""Attention over a paged cache where rows see nothing, and where queries, keys or values are not
finite, in every form that the kernel takes: rows four times in a tile (many items of up to 16
rows), one row tile, pairs of row tiles (more than 128 rows), items of one CTA and shared ones.
The formulas, the cache and the tolerances are those of test_paged_attention."""
import math

import pytest
import torch

import oracle
from test_paged_attention import Cache, _tree

# (sequences, query heads, key/value heads, tokens, head dim, lengths): what the rows and items give
FORMS = {
    "quad": (60, 4, 1, 2, 64, [5 + 7 * i for i in range(60)]),              # eight rows, items of one CTA and shared ones
    "split": (2, 8, 2, 5, 64, [90, 40]),                                    # 20 rows, items of one tile
    "split shared": (1, 8, 2, 5, 128, [3000]),
    "pair": (2, 8, 2, 40, 64, [70, 0]),                                     # 160 rows, items of one tile
    "pair shared": (1, 8, 2, 70, 128, [1500]),
}


def _cache(form, dtype, seed=0):
    b, hq, hkv, t, d, lens = FORMS[form]
    return Cache(b, hq, hkv, t, d, dtype, 16, lens, seed=seed)


def _slot(c, b, at):
    """Index of token `at` of sequence b in a cache, all heads."""
    return int(c.table[b, at // 16]), slice(None), at % 16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,hq,hkv,t,lens", [
    (2, 8, 2, 40, [0, 200]),            # 160 rows over an empty cache: an item of one tile, one CTA's
    (90, 8, 2, 40, [0] * 90),           # more items than CTAs
    (1, 2, 1, 300, [0]),                # items of three tiles that CTAs share
    (2, 256, 2, 2, [0, 50])])           # a token's 128 heads fill a row tile
def test_rows_that_see_nothing_among_more_than_128(dtype, b, hq, hkv, t, lens, device_ok):
    c = Cache(b, hq, hkv, t, 64, dtype, 16, lens, seed=t)
    mask = torch.rand(t, t, generator=torch.Generator().manual_seed(1)).cuda() < 0.2
    mask[0] = mask[t // 2] = False
    got = c.run(tree_mask=mask)
    c.check(got, mask)
    assert bool((got[0, :, [0, t // 2]] == 0).all())
    none = torch.zeros_like(mask)
    got = c.run(tree_mask=none)
    c.check(got, none)
    assert bool((got[0] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_large_values_stay_with_the_rows_that_see_them(form, device_ok):
    # 2^118 times 2^-125 would be a 2^-7: a masked draft's weight is zero
    c, clean = _cache(form, torch.bfloat16), _cache(form, torch.bfloat16)
    t = c.q.shape[2]
    mask = torch.eye(t, dtype=torch.bool, device="cuda")
    mask[:, 0] = True
    for b in range(c.q.shape[0]):
        for j in range(1, t):
            c.vc[_slot(c, b, int(c.lens[b]) + j)] = 2.0 ** 118
    got = c.run(tree_mask=mask)
    c.check(got, mask)
    assert torch.equal(got[:, :, 0], clean.run(tree_mask=mask)[:, :, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("residue", range(8))
def test_a_key_of_nan_reaches_every_row_that_sees_it(form, draft, residue, device_ok):
    # at every place of the eight scores that one round of exponentials takes
    c = _cache(form, torch.bfloat16)
    b, t = c.q.shape[0], c.q.shape[2]
    mask = _tree(b, t, seed=residue)
    for i in range(b):
        have = int(c.lens[i])
        first, end = (have, have + t) if draft else (0, have)
        places = [at for at in range(first, end) if at % 8 == residue]
        if places:
            c.kc[_slot(c, i, places[len(places) // 2])][..., 3] = math.nan
    got = c.run(tree_mask=mask)
    want, _ = oracle.paged_attention_ref(c.q, c.kc, c.vc, c.table, c.lens, None, mask)
    assert torch.equal(torch.isnan(got), torch.isnan(want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form", FORMS)
def test_a_query_of_nan_gives_a_row_of_nan(dtype, form, device_ok):
    c, clean = _cache(form, dtype), _cache(form, dtype)
    t = c.q.shape[2]
    c.q[:, 1, t - 1, 5] = math.nan
    got = c.run()
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[:, 1, t - 1] = True
    assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[~bad], clean.run()[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("first,end", [(0, 5), (0, 32), (32, 64), (0, 128), (128, 1400)])
def test_ranges_of_nan_keys_are_not_dropped(form, first, end, device_ok):
    # a quarter of a tile, a tile, a CTA's whole range: states whose scores are all NaN
    c = _cache(form, torch.bfloat16)
    for i in range(c.q.shape[0]):
        for at in range(first, min(end, int(c.lens[i]))):
            c.kc[_slot(c, i, at)] = math.nan
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_scores_of_minus_infinity(form, device_ok):
    # a key of -inf has no weight; where a row sees no other, its softmax is 0 / 0.  A row that sees
    # no key at all stays zero.
    c = _cache(form, torch.bfloat16)
    b, t = c.q.shape[0], c.q.shape[2]
    c.q[..., 0] = 1.0
    mask = _tree(b, t, seed=2)
    for i in range(b):
        for at in range(int(c.lens[i])):
            if i % 2 == 0 or at % 3 == 0:
                c.kc[_slot(c, i, at)][..., 0] = -math.inf
        c.kc[_slot(c, i, int(c.lens[i]) + t - 1)][..., 0] = -math.inf
    c.check(c.run(tree_mask=mask), mask)
    mask[:, t - 1] = False
    mask[:, t - 2] = False
    mask[:, t - 2, t - 1] = True                 # sees the draft of -inf alone, besides the cache
    got = c.run(tree_mask=mask)
    c.check(got, mask)
    for i in range(b):
        if int(c.lens[i]) == 0:
            assert bool((got[i, :, t - 1] == 0).all()) and bool(torch.isnan(got[i, :, t - 2]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_a_query_of_infinity(form, device_ok):
    # scores of inf make the row NaN, scores of -inf drop the key
    c, clean = _cache(form, torch.bfloat16), _cache(form, torch.bfloat16)
    t = c.q.shape[2]
    c.q[:, 1, t - 1, 5] = math.inf
    got = c.run()
    want, _ = oracle.paged_attention_ref(c.q, c.kc, c.vc, c.table, c.lens)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[:, 1, t - 1] = False
    assert torch.equal(got[rest], clean.run()[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_draft_values_that_are_not_finite_change_their_columns_alone(dtype, form, value, device_ok):
    c, clean = _cache(form, dtype), _cache(form, dtype)
    b, t = c.q.shape[0], c.q.shape[2]
    bad = ((1, 5), (t // 2, 33), (t - 1, 5))
    for i in range(b):
        for j, column in bad:
            c.vc[_slot(c, i, int(c.lens[i]) + j)][..., column] = value
    causal = torch.ones(b, t, t, dtype=torch.bool, device="cuda").tril()
    for mask in (_tree(b, t, seed=3), None):
        sees = causal if mask is None else mask
        where = torch.zeros_like(c.q, dtype=torch.bool)
        for j, column in bad:
            where[..., column] |= sees[:, None, :, j]
        got, want = c.run(tree_mask=mask), clean.run(tree_mask=mask)
        clean.check(want, mask)
        assert torch.equal(got[~where], want[~where])
        assert bool((torch.isnan(got[where]) if math.isnan(value) else got[where] == value).all())


@pytest.mark.gpu
@pytest.mark.parametrize("columns", [[7], list(range(64))])
def test_a_chunk_whose_values_are_all_nan(columns, device_ok):
    # as after a failure in the layer before: the call ends in good time and says NaN
    b, t, have = 2, 1500, [0, 333]
    c, clean = (Cache(b, 4, 2, t, 64, torch.bfloat16, 16, have) for _ in range(2))
    for i in range(b):
        at = torch.arange(have[i] + 20, have[i] + t, device="cuda")
        rows = c.vc[c.table[i].long()[at // 16], :, at % 16]
        rows[..., columns] = math.nan
        c.vc[c.table[i].long()[at // 16], :, at % 16] = rows
    got, want = c.run(), clean.run()
    where = torch.zeros_like(got, dtype=torch.bool)
    where[:, :, 20:, columns] = True
    assert torch.equal(torch.isnan(got), where)
    assert torch.equal(got[~where], want[~where])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("form", FORMS)
def test_values_of_earlier_tokens_that_are_not_finite(dtype, form, device_ok):
    # column 3: inf, 4: -inf, 5: both, 6: NaN and inf, 40: NaN; the last at the last earlier token
    c = _cache(form, dtype)
    for i in range(c.q.shape[0]):
        have = int(c.lens[i])
        for column, at, value in ((3, 0, math.inf), (4, have // 2, -math.inf), (5, 1, math.inf), (5, have - 2, -math.inf),
                                  (6, 2, math.nan), (6, 3, math.inf), (40, have - 1, math.nan)):
            if have > 4:
                c.vc[_slot(c, i, at)][..., column] = value
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("b", [2, 60])
def test_a_decode_step_whose_own_value_is_not_finite(b, value, device_ok):
    c = Cache(b, 4, 1, 1, 64, torch.bfloat16, 16, [3 * i for i in range(b)])
    for i in range(b):
        c.vc[_slot(c, i, 3 * i)][..., i % 64] = value
    c.check(c.run())

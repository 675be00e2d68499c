"""Attention of a step's tokens over a paged cache against 64-bit formulas.

Tolerance of an output value: half a step of its type, u, and, relative to the magnitude
mag = sum_p softmax_p |v_p|,
  * u for the weights, which are rounded to the inputs' type before they multiply V;
  * 2 d for an error d of a score (a weight and the sum it is divided by may err oppositely):
    d = D * 2^-23 * scale * max |q| max |k| for the fp32 sum of D products (one step per addition,
    tensor cores may truncate), and 2^-20 for the exponent's own rounding and exp2;
  * float16 weights below 2^-14 lose up to 2^-25 absolute, keys times, against a sum of at least
    one, times the largest |v|.
"""
import ctypes
import math

import pytest
import torch

import b200k
import oracle
from b200k import _lib


class Cache:
    """Queries of a step over a cache with its pages in no order.  Everything that is not a token
    of some sequence is NaN, in K and in V: pages of no sequence and slots behind the last one."""

    def __init__(self, b, hq, hkv, t, d, dtype, page, lens, new=None, slots_first=False, seed=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.q = torch.randn(b, t, hq, d, generator=g).to(dtype).cuda().transpose(1, 2) * spread
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.new = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
        fresh = [t] * b if new is None else [max(0, min(n, t)) for n in new]
        per = max(1, max((n + t + page - 1) // page for n in lens))
        pages = b * per + 3
        self.table = torch.randperm(pages, generator=g)[:b * per].reshape(b, per).int().cuda()
        shape = (pages, page, hkv, d) if slots_first else (pages, hkv, page, d)
        self.kc, self.vc = (torch.full(shape, math.nan, dtype=dtype, device="cuda") for _ in range(2))
        if slots_first:
            self.kc, self.vc = self.kc.transpose(1, 2), self.vc.transpose(1, 2)
        for i, (have, n) in enumerate(zip(lens, fresh)):
            if n:
                at = torch.arange(have + n, device="cuda")
                where = self.table[i].long()[at // page]
                for c in (self.kc, self.vc):
                    c[where, :, at % page] = torch.randn(have + n, hkv, d, generator=g).to(dtype).cuda()
        self.real = torch.arange(t, device="cuda") < torch.tensor(fresh, device="cuda")[:, None]

    def run(self, **kw):
        return b200k.paged_attention(self.q, self.kc, self.vc, self.table, self.lens, new_lens=self.new, **kw)

    def check(self, got, mask=None, scale=None):
        d = self.q.shape[3]
        s = scale or 1.0 / math.sqrt(d)
        want, mag = oracle.paged_attention_ref(self.q, self.kc, self.vc, self.table, self.lens, self.new, mask, scale)
        u = torch.finfo(got.dtype).eps / 2
        kn = self.kc.double().nan_to_num(0, 0, 0).norm(dim=-1).max()
        err_score = d * 2.0 ** -23 * s * float(self.q.double().norm(dim=-1).max() * kn) + 2.0 ** -20
        bound = u * want.abs() + (u + 2 * err_score) * mag
        if got.dtype == torch.float16:
            keys = int(self.lens.max()) + self.q.shape[2]
            bound += keys * 2.0 ** -25 * float(self.vc.double().nan_to_num(0, 0, 0).abs().max()) + 2.0 ** -25
        assert got.dtype == self.q.dtype and got.shape == self.q.shape
        real = self.real[:, None, :, None].expand_as(want)
        assert torch.equal(torch.isnan(got[real]), torch.isnan(want[real]))
        good = real & torch.isfinite(want)
        inf = real & torch.isinf(want)
        assert torch.equal(got[inf].double(), want[inf])
        err = (got.double() - want).abs()
        assert bool((err[good] <= bound[good]).all()), (
            f"{int((err[good] > bound[good]).sum())} values off, worst {float((err[good] / bound[good]).max()):.3g} bounds")
        return want


def _tree(b, t, seed=0):
    """Ancestors and self, every drafted token hanging from an earlier one."""
    g = torch.Generator().manual_seed(seed)
    sees = torch.eye(t, dtype=torch.bool).repeat(b, 1, 1)
    for i in range(b):
        for j in range(1, t):
            sees[i, j] |= sees[i, int(torch.randint(0, j, (1,), generator=g))]
    return sees.cuda()


# ---- without a GPU -------------------------------------------------------------------------------

def test_refusals_of_the_entry_point():
    h = _lib.lib()
    assert h.b200k_paged_attention(None, None) == _lib.INVALID_ARG
    assert h.b200k_paged_attention_workspace_bytes(None) == 0

    def call(**change):
        a = _lib.PagedAttentionArgs()
        a.batch, a.tokens, a.heads_q, a.heads_kv, a.head_dim = 1, 4, 4, 2, 64
        a.dtype, a.page_size, a.num_pages, a.max_pages, a.qk_scale = _lib.BF16, 16, 8, 4, 0.125
        a.q = a.k_cache = a.v_cache = a.out = a.page_table = a.cache_lens = 1 << 20
        a.kc_stride_p = a.vc_stride_p = 2048
        a.kc_stride_h = a.vc_stride_h = 1024
        a.kc_stride_s = a.vc_stride_s = 64
        for name, value in change.items():
            setattr(a, name, value)
        return h.b200k_paged_attention(ctypes.byref(a), None)

    assert call(heads_q=5) == _lib.INVALID_ARG
    assert call(heads_kv=0) == _lib.INVALID_ARG
    assert call(dtype=_lib.F32) == _lib.INVALID_ARG
    assert call(head_dim=136) == _lib.UNSUPPORTED
    assert call(head_dim=60) == _lib.UNSUPPORTED
    assert call(page_size=12) == _lib.UNSUPPORTED
    assert call(page_size=0) == _lib.UNSUPPORTED
    assert call(max_pages=1 << 30) == _lib.UNSUPPORTED
    assert call(batch=1 << 20) == _lib.UNSUPPORTED
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert call(qk_scale=scale) == _lib.INVALID_ARG
    assert call(q=None) == _lib.INVALID_ARG
    assert call(page_table=None) == _lib.INVALID_ARG
    assert call(heads_q=258) == _lib.UNSUPPORTED
    assert call(kc_stride_s=60) == _lib.UNSUPPORTED
    assert call(q_stride_t=60) == _lib.UNSUPPORTED
    assert call(v_cache=(1 << 20) + 8) == _lib.UNSUPPORTED
    assert call(num_pages=0) == _lib.INVALID_ARG
    assert call(tokens=0, q=None) == _lib.OK


def test_scales_whose_product_with_log2_e_is_infinite_are_refused():
    a = _lib.PagedAttentionArgs()
    a.batch, a.tokens, a.heads_q, a.heads_kv, a.head_dim = 1, 4, 4, 2, 64
    a.dtype, a.page_size, a.max_pages = _lib.BF16, 16, 4
    a.q = a.k_cache = a.v_cache = a.out = a.page_table = a.cache_lens = 1 << 20
    for scale, message in ((2.0e38, b"no pages"), (2.4e38, b"qk_scale"), (2.9e38, b"qk_scale")):
        a.qk_scale = scale
        assert _lib.lib().b200k_paged_attention(ctypes.byref(a), None) == _lib.INVALID_ARG
        assert message in _lib.lib().b200k_last_error()


def test_the_limit_of_key_tiles_counts_full_tables():
    h = _lib.lib()

    def call(**change):
        a = _lib.PagedAttentionArgs()
        a.batch, a.tokens, a.heads_q, a.heads_kv, a.head_dim = 512, 2048, 32, 8, 128
        a.dtype, a.page_size, a.max_pages, a.qk_scale = _lib.BF16, 16, 1 << 16, 0.125
        a.q = a.k_cache = a.v_cache = a.out = a.page_table = a.cache_lens = 1 << 20
        for name, value in change.items():
            setattr(a, name, value)
        return h.b200k_paged_attention(ctypes.byref(a), None)

    # 512 x 8 items of 32 row tiles, tables of 2^20 tokens: 2^30 (refused for its lack of pages)
    assert call() == _lib.INVALID_ARG
    assert call(batch=1023) == _lib.INVALID_ARG
    assert call(batch=1024) == _lib.UNSUPPORTED                       # 2^31
    assert call(tokens=1 << 62, heads_q=8) == _lib.UNSUPPORTED        # counts whose product is no 64-bit number
    assert call(tokens=1 << 14, batch=65535, page_size=8, max_pages=1 << 26) == _lib.UNSUPPORTED


def test_refusals_of_the_wrapper():
    q = torch.zeros(1, 2, 3, 64).half()
    cache = torch.zeros(4, 2, 16, 64).half()
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        b200k.paged_attention(q, cache, cache, table, lens)
    with pytest.raises(ValueError, match="4D"):
        b200k.paged_attention(q[0], cache, cache, table, lens)


# ---- on the GPU ----------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("slots_first", [False, True])
@pytest.mark.parametrize("b,hq,hkv,t,d,page,lens,new,tree", [
    (1, 1, 1, 1, 64, 8, [0], None, False),                            # the first token: it sees itself
    (1, 4, 1, 1, 128, 16, [1023], None, False),                       # a whole number of key tiles
    (3, 8, 2, 1, 128, 16, [127, 128, 129], None, False),
    (5, 8, 2, 1, 128, 32, [0, 5000, 3, 700, 64], [1, 1, 0, 1, 1], False),
    (4, 8, 8, 5, 64, 24, [0, 100, 125, 300], [5, 1, 4, 0], False),    # pages that end inside a tile
    (2, 32, 8, 16, 128, 16, [250, 1000], [16, 9], True),              # 64 rows
    (3, 6, 2, 7, 96, 40, [10, 377, 0], [7, 7, 3], True),              # a padded head, an odd group
    (2, 8, 1, 40, 128, 128, [129, 511], [40, 33], True),              # 320 rows: three row tiles
    (1, 4, 2, 200, 128, 64, [300], None, False),                      # a chunk of a prompt
    (2, 2, 2, 300, 64, 16, [0, 77], [300, 129], False),
    (2, 3, 3, 2, 8, 8, [9, 0], None, True),
    (1, 5, 1, 3, 72, 56, [99], [3], True)])
def test_matches_the_formula(dtype, slots_first, b, hq, hkv, t, d, page, lens, new, tree, device_ok):
    c = Cache(b, hq, hkv, t, d, dtype, page, lens, new, slots_first, seed=t + d)
    mask = _tree(b, t) if tree else None
    got = c.run(tree_mask=mask)
    c.check(got, mask)
    assert bool((got.transpose(1, 2)[~c.real] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("hkv,lens", [(1, [40000]), (2, [33000, 5]), (8, [9000])])
def test_long_sequences_shared_by_many_ctas(hkv, lens, device_ok):
    c = Cache(len(lens), 4 * hkv, hkv, 1, 128, torch.bfloat16, 64, lens)
    c.check(c.run())


@pytest.mark.gpu
def test_many_short_sequences(device_ok):
    # more sequences than a warp has lanes, a third of them empty
    g = torch.Generator().manual_seed(2)
    lens = torch.randint(0, 400, (75,), generator=g).tolist()
    new = torch.randint(0, 4, (75,), generator=g).tolist()
    c = Cache(75, 4, 2, 3, 64, torch.float16, 16, lens, new)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("b,hq,hkv,t,d,lens,tree", [
    (16, 32, 8, 1, 128, [3333 + 67 * i for i in range(16)], False),     # a dozen tiles a CTA
    (12, 8, 2, 16, 128, [5000 + 131 * i for i in range(12)], True),
    (9, 8, 2, 60, 64, [4100 - 77 * i for i in range(9)], True)])        # two row tiles
def test_many_tiles_in_a_row(b, hq, hkv, t, d, lens, tree, device_ok):
    # long runs inside one CTA: the last tile's rows of V are cleared only after the tile before
    # has been used
    c = Cache(b, hq, hkv, t, d, torch.bfloat16, 32, lens)
    mask = _tree(b, t) if tree else None
    first = c.run(tree_mask=mask)
    c.check(first, mask)
    for _ in range(3):
        assert torch.equal(c.run(tree_mask=mask), first)


@pytest.mark.gpu
@pytest.mark.parametrize("b,hq,hkv,t,d,lens,new", [
    (2, 6, 2, 60, 64, [500, 37], [60, 50]),      # three heads a token: halves of 126 rows
    (1, 7, 1, 40, 128, [300], None),             # halves of 18 tokens, 126 rows
    (2, 128, 1, 2, 64, [200, 0], [1, 2]),        # a token's heads fill a half
    (1, 100, 1, 3, 128, [130], None),            # 100 of 128 rows a half, the last half empty
    (1, 10, 5, 64, 96, [1000], None)])
def test_row_tiles_of_whole_tokens(b, hq, hkv, t, d, lens, new, device_ok):
    c = Cache(b, hq, hkv, t, d, torch.bfloat16, 16, lens, new)
    for mask in (None, _tree(b, t, seed=3)):
        c.check(c.run(tree_mask=mask), mask)
    c.q = c.q[:1].expand(b, hq, t, d) if b > 1 else c.q
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,hq,hkv,t,d,page,longest,tree", [
    (50, 1, 1, 1, 128, 16, 300, False),          # one row an item, several items a CTA
    (25, 6, 2, 5, 96, 24, 700, True),            # 15 rows
    (17, 12, 3, 4, 72, 8, 90, True),             # 16 rows, items of one tile
    (13, 16, 4, 3, 8, 16, 1500, True),
    (100, 8, 1, 2, 64, 16, 130, False),          # 16 rows, a tile or two
    (70, 17, 1, 1, 128, 32, 260, False)])        # 17 rows: the tile is not shared by four copies
def test_many_items_with_few_rows(dtype, b, hq, hkv, t, d, page, longest, tree, device_ok):
    g = torch.Generator().manual_seed(b)
    lens = torch.randint(0, longest + 1, (b,), generator=g).tolist()
    new = torch.randint(0, t + 1, (b,), generator=g).tolist()
    lens[0], new[0] = longest, t
    c = Cache(b, hq, hkv, t, d, dtype, page, lens, new, seed=b)
    mask = _tree(b, t) if tree else None
    got = c.run(tree_mask=mask)
    c.check(got, mask)
    assert torch.equal(got, c.run(tree_mask=mask))
    assert bool((got.transpose(1, 2)[~c.real] == 0).all())
    if t > 1:                                     # rows that see nothing, or only what was there
        none = torch.zeros(t, t, dtype=torch.bool, device="cuda")
        c.check(c.run(tree_mask=none), none)
    out = torch.full_like(got, 7.0)
    c.run(tree_mask=mask, out=out)
    assert bool((out.transpose(1, 2)[~c.real] == 7).all())
    real = c.real[:, None, :, None].expand_as(got)
    assert torch.equal(out[real], got[real])


@pytest.mark.gpu
@pytest.mark.parametrize("t,hq", [(1, 64), (3, 128)])
def test_more_items_than_a_grid_has_rows(t, hq, device_ok):
    g = torch.Generator().manual_seed(t)
    b = 1100
    lens = torch.randint(0, 31, (b,), generator=g).tolist()
    c = Cache(b, hq, 64, t, 8, torch.bfloat16, 8, lens, torch.randint(0, t + 1, (b,), generator=g).tolist())
    got = c.run()
    c.check(got)
    assert bool((got.transpose(1, 2)[~c.real] == 0).all())


@pytest.mark.gpu
def test_wide_tables_with_many_row_tiles(device_ok):
    # 8 x 4 items of 9 row tiles, tables of 2^29 tokens: more than 2^30 key tiles, were they full
    c = Cache(8, 16, 4, 520, 8, torch.bfloat16, 4096, [0, 3, 900, 77, 128, 2000, 5, 4090])
    want = c.run()
    table = torch.zeros(8, 1 << 17, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table
    c.table = table
    got = c.run()
    c.check(got)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [math.nan, -math.inf])
def test_many_items_keep_values_that_are_not_finite_to_their_rows(value, device_ok):
    # every sequence has a draft with such a value, at every place in a tile; queries that see it not
    # stay finite, the others have it in that column alone
    b, t = 60, 4
    c = Cache(b, 2, 1, t, 64, torch.bfloat16, 16, [3 + 7 * i for i in range(b)], seed=5)
    mask = torch.tensor([[1, 0, 0, 0], [1, 1, 0, 0], [1, 0, 1, 0], [1, 0, 1, 1]], device="cuda").bool()
    for i in range(b):
        at = 3 + 7 * i + 1                       # draft 1: only query 1 sees it
        c.vc[int(c.table[i, at // 16]), 0, at % 16, 5] = value
    got = c.run(tree_mask=mask)
    seen = [0, 2, 3]
    assert bool(torch.isfinite(got[:, :, seen]).all())
    assert not bool(torch.isfinite(got[:, :, 1, 5]).any())
    rest = [i for i in range(64) if i != 5]
    assert bool(torch.isfinite(got[:, :, 1][..., rest]).all())
    clean = Cache(b, 2, 1, t, 64, torch.bfloat16, 16, [3 + 7 * i for i in range(b)], seed=5)
    want = clean.run(tree_mask=mask)
    assert torch.equal(got[:, :, seen], want[:, :, seen])
    # the same sums, one weight kept in fp32 instead of bfloat16: 2^-8 of it times |v| < 5
    assert float((got[:, :, 1][..., rest].double() - want[:, :, 1][..., rest].double()).abs().max()) <= 2 * 5 * 2.0 ** -8


@pytest.mark.gpu
def test_many_items_with_scores_that_grow(device_ok):
    lens = [900 - 11 * i for i in range(60)]
    c = Cache(60, 4, 1, 2, 128, torch.bfloat16, 16, lens, spread=4.0)
    for i, have in enumerate(lens):
        at = torch.arange(have + 2, device="cuda")
        where = c.table[i].long()[at // 16]
        ramp = torch.linspace(0.1, 5.0, have + 2, device="cuda").roll(have // 3)[:, None, None]
        c.kc[where, :, at % 16] = (c.kc[where, :, at % 16] * ramp).bfloat16()
    c.check(c.run())


@pytest.mark.gpu
def test_masks_that_leave_rows_empty(device_ok):
    for lens in ([0, 0], [0, 200]):
        c = Cache(2, 4, 2, 6, 64, torch.bfloat16, 16, lens)
        mask = torch.rand(6, 6, generator=torch.Generator().manual_seed(1)).cuda() < 0.4
        mask[2] = False
        got = c.run(tree_mask=mask)
        c.check(got, mask)
        assert bool((got[0, :, 2] == 0).all())
        got = c.run(tree_mask=torch.zeros_like(mask))
        c.check(got, torch.zeros_like(mask))
        assert bool((got[0] == 0).all())


@pytest.mark.gpu
def test_masks_through_strides(device_ok):
    c = Cache(2, 4, 2, 6, 64, torch.bfloat16, 16, [30, 100])
    mask = _tree(2, 6)
    want = c.run(tree_mask=mask)
    wide = torch.zeros(2, 6, 13, dtype=torch.bool, device="cuda")
    wide[..., 1::2] = mask
    assert torch.equal(c.run(tree_mask=wide[..., 1::2]), want)
    assert torch.equal(c.run(tree_mask=mask.transpose(1, 2).contiguous().transpose(1, 2)), want)
    assert torch.equal(c.run(tree_mask=mask[:1].expand(2, 6, 6)), c.run(tree_mask=mask[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("have", [3, 126, 700])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_drafts_that_are_not_finite_reach_only_those_who_see_them(dtype, have, value, device_ok):
    c = Cache(1, 4, 2, 5, 64, dtype, 16, [have], seed=have)
    mask = _tree(1, 5, seed=1)
    mask[0, 2:, 1] = False
    mask[0, 4, 3] = False
    for draft, cache in ((1, c.vc), (3, c.kc)):
        at = have + draft
        cache[int(c.table[0, at // 16]), 0, at % 16, 5] = value
    got = c.run(tree_mask=mask)
    want, _ = oracle.paged_attention_ref(c.q, c.kc, c.vc, c.table, c.lens, None, mask)
    clean = torch.tensor([True, False, True, False, True], device="cuda")     # who sees neither 1 nor 3
    assert bool(torch.isfinite(got[:, :, clean]).all()) and bool(torch.isfinite(got[:, 2:]).all())
    assert torch.equal(got[0, :2, 1, 5].double(), want[0, :2, 1, 5]) or math.isnan(value)
    assert not bool(torch.isfinite(got[0, :2, 1, 5]).any())
    # the same row's other columns are the formula's too (NaN keys make whole rows NaN: query 3)
    rest = [i for i in range(64) if i != 5]
    seen = [0, 1, 2, 4]
    err = (got[:, :, seen][..., rest].double() - want[:, :, seen][..., rest]).abs()
    # |v| < 5, |q| |k| < 15 * 15: the module's tolerance with mag and the output below 5
    u = torch.finfo(dtype).eps / 2
    assert float(err.max()) <= 5 * (2 * u + 2 * (64 * 2.0 ** -23 * 0.125 * 225 + 2.0 ** -20)) + (have + 5) * 2.0 ** -25 * 5


@pytest.mark.gpu
def test_scores_that_grow_along_the_keys(device_ok):
    # the running maximum rises by far more than the deferred rescale's threshold, and falls off
    c = Cache(2, 4, 2, 3, 128, torch.bfloat16, 16, [3000, 700], spread=4.0)
    for i, have in enumerate((3000, 700)):
        at = torch.arange(have + 3, device="cuda")
        ramp = torch.linspace(0.1, 5.0, have + 3, device="cuda").roll(have // 3)[:, None, None]
        where = c.table[i].long()[at // 16]
        c.kc[where, :, at % 16] = (c.kc[where, :, at % 16] * ramp).bfloat16()
    c.check(c.run())
    c.check(c.run(qk_scale=0.5), scale=0.5)


@pytest.mark.gpu
def test_padding_rows_of_a_given_output_stay(device_ok):
    c = Cache(3, 4, 2, 6, 128, torch.bfloat16, 16, [12, 90, 40], [6, 2, 0])
    out = torch.full((3, 4, 6, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    assert c.run(out=out) is out
    c.check(out)
    assert bool((out.transpose(1, 2)[~c.real] == 7).all())
    # an output in (B, T, H, D) storage and one whose rows start off 16-byte boundaries
    side = torch.zeros(3, 6, 4, 128, dtype=torch.bfloat16, device="cuda")
    c.run(out=side.transpose(1, 2))
    c.check(side.transpose(1, 2))
    odd = torch.full((3, 4, 6, 131), 5.0, dtype=torch.bfloat16, device="cuda")
    c.run(out=odd[..., 3:])
    c.check(odd[..., 3:])
    assert bool((odd[..., :3] == 5).all())
    c.q = torch.randn(3, 4, 6, 129, device="cuda").bfloat16()[..., 1:]       # queries likewise
    c.check(c.run())
    c.q = torch.randn(3, 4, 128, 6, device="cuda").bfloat16().transpose(2, 3)
    c.check(c.run())


@pytest.mark.gpu
def test_agrees_with_contiguous_attention(device_ok):
    # the same keys as one contiguous (B, H, S, D) tensor through cutile_fmha
    have, t = 700, 5
    c = Cache(2, 8, 2, t, 128, torch.bfloat16, 16, [have, have])
    at = torch.arange(have + t, device="cuda")
    k, v = (torch.stack([x[c.table[i].long()[at // 16], :, at % 16] for i in range(2)]).transpose(1, 2).contiguous()
            for x in (c.kc, c.vc))
    ref = b200k.cutile_fmha(c.q.contiguous(), k, v, causal=True, input_pos=have, query_group_size=4)
    torch.testing.assert_close(c.run().float(), ref.float(), atol=1e-2, rtol=5e-2)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [1, 5])
def test_sequences_share_the_pages_of_a_prefix(t, device_ok):
    c = Cache(6, 8, 2, t, 128, torch.bfloat16, 16, [640, 647, 655, 900, 640, 1300])
    c.table[1:, :40] = c.table[0, :40]            # 640 tokens, whole pages
    c.check(c.run())
    c.table[4] = c.table[0]                       # a whole sequence twice, its step's tokens too
    got = c.run()
    c.check(got)
    assert torch.equal(got, c.run())


@pytest.mark.gpu
def test_pages_and_lengths_out_of_range_are_reported():
    c = Cache(3, 4, 2, 2, 64, torch.bfloat16, 16, [100, 50, 200])
    good = c.run()
    torch.cuda.synchronize()
    b200k.raise_on_device_error()
    for page in (-1, c.kc.shape[0], 2 ** 31 - 1, -2 ** 31):
        table = c.table.clone()
        table[1, 2] = page
        got = b200k.paged_attention(c.q, c.kc, c.vc, table, c.lens)
        assert torch.equal(got[0], good[0]) and torch.equal(got[2], good[2])
        with pytest.raises(b200k.B200KError, match="page of sequence 1"):
            b200k.raise_on_device_error()
    for have in (-5, 10 ** 6, 2 ** 31 - 1):
        lens = c.lens.clone()
        lens[1] = have
        got = b200k.paged_attention(c.q, c.kc, c.vc, c.table, lens)
        torch.testing.assert_close(got[0].float(), good[0].float(), atol=1e-2, rtol=5e-2)
        with pytest.raises(b200k.B200KError, match="page of sequence 1"):
            b200k.raise_on_device_error()
    b200k.raise_on_device_error()


@pytest.mark.gpu
def test_offsets_beyond_32_bits(device_ok):
    page, hkv, d = 128, 8, 128
    pages = (1 << 31) // (page * hkv * d) + 4
    c = Cache(1, 8, 8, 1, d, torch.float16, page, [200])
    kc, vc = (torch.zeros(pages, hkv, page, d, dtype=torch.float16, device="cuda") for _ in range(2))
    for i in range(2):
        kc[pages - 1 - i], vc[pages - 1 - i] = c.kc[int(c.table[0, i])], c.vc[int(c.table[0, i])]
    c.kc, c.vc = kc, vc
    c.table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    got = c.run()
    c.kc, c.vc = kc[-4:].clone(), vc[-4:].clone()
    c.table = torch.tensor([[3, 2]], dtype=torch.int32, device="cuda")
    c.check(got)


@pytest.mark.gpu
def test_empty_calls(device_ok):
    c = Cache(2, 4, 2, 3, 64, torch.float16, 16, [5, 9])
    assert b200k.paged_attention(c.q[:, :, :0], c.kc, c.vc, c.table, c.lens).shape == (2, 4, 0, 64)
    assert b200k.paged_attention(c.q[:0], c.kc, c.vc, c.table[:0], c.lens[:0]).shape == (0, 4, 3, 64)
    none = b200k.paged_attention(c.q, c.kc, c.vc, c.table, c.lens, new_lens=torch.zeros_like(c.lens))
    assert bool((none == 0).all())


@pytest.mark.gpu
def test_refused_inputs(device_ok):
    c = Cache(2, 4, 2, 3, 64, torch.bfloat16, 16, [5, 9])

    def call(q=c.q, kc=c.kc, vc=c.vc, table=c.table, lens=c.lens, **kw):
        return b200k.paged_attention(q, kc, vc, table, lens, **kw)

    with pytest.raises(TypeError, match="float16 and bfloat16"):
        call(q=c.q.float())
    with pytest.raises(ValueError, match="multiple of the cache's heads"):
        call(q=c.q[:, :3])
    with pytest.raises(ValueError, match="data type"):
        call(q=c.q.half())
    with pytest.raises(ValueError, match="multiple of 8 tokens"):
        call(kc=c.kc[:, :, :12], vc=c.vc[:, :, :12])
    with pytest.raises(ValueError, match="16-byte"):
        wide = torch.zeros(4, 2, 16, 68, dtype=torch.bfloat16, device="cuda")[..., :64]
        call(kc=wide, vc=wide)
    with pytest.raises(ValueError, match="at most 128 query heads"):
        call(q=torch.zeros(2, 258, 3, 64, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(ValueError, match="multiple of 8 up to 128"):
        big = torch.zeros(4, 2, 16, 136, dtype=torch.bfloat16, device="cuda")
        call(q=torch.zeros(2, 4, 3, 136, dtype=torch.bfloat16, device="cuda"), kc=big, vc=big)
    with pytest.raises(TypeError, match="bool"):
        call(tree_mask=torch.ones(3, 3, device="cuda"))
    with pytest.raises(ValueError, match="tree_mask must be"):
        call(tree_mask=torch.ones(2, 2, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError, match="device"):
        call(tree_mask=torch.ones(3, 3, dtype=torch.bool))
    for scale in (0.0, -0.1, math.nan, math.inf):
        with pytest.raises(ValueError, match="qk_scale"):
            call(qk_scale=scale)
    with pytest.raises(TypeError, match="int32"):
        call(lens=c.lens.long())
    with pytest.raises(ValueError, match="autograd"):
        call(q=c.q.clone().requires_grad_())
    with pytest.raises(ValueError, match="out must have"):
        call(out=torch.empty(2, 4, 3, 32, dtype=torch.bfloat16, device="cuda"))


@pytest.mark.gpu
def test_captured_replayed_and_on_two_streams(device_ok):
    c = Cache(3, 8, 2, 4, 128, torch.bfloat16, 16, [500, 90, 1500], [4, 2, 3])
    mask = _tree(3, 4)
    c.run(tree_mask=mask)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(c.run(tree_mask=mask))
        graphs.append(g)
    first = c.q.clone()
    for _ in range(2):
        c.q.normal_()
        c.lens -= 7                                   # other lengths: another split of the work
        graphs[0].replay()
        one = outs[0].clone()
        graphs[1].replay()
        torch.cuda.synchronize()
        c.check(one, mask)
        assert torch.equal(one, outs[1]) and torch.equal(one, c.run(tree_mask=mask))
    c.q.copy_(first)
    want = c.run(tree_mask=mask)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got += [c.run(tree_mask=mask) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.gpu
def test_captured_behind_other_kinds_of_work(device_ok):
    # behind a copy, behind a join of two streams, and one call right behind another
    c = Cache(2, 8, 2, 3, 128, torch.bfloat16, 16, [500, 90])
    src, side = torch.randn_like(c.q), torch.cuda.Stream()
    c.run()
    torch.cuda.synchronize()
    q = c.q
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.q = q.clone(memory_format=torch.contiguous_format)
        c.q.copy_(src)
        one = c.run()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = c.kc * 1
        c.q = c.q + 0
        torch.cuda.current_stream().wait_stream(side)
        two = c.run()
        again = [c.run() for _ in range(4)][-1]
    for _ in range(2):
        src.normal_()
        graph.replay()
        torch.cuda.synchronize()
        c.q = src
        want = c.run()
        c.check(want)
        assert torch.equal(one, want) and torch.equal(two, want) and torch.equal(again, want)
    assert other.shape == c.kc.shape


@pytest.mark.gpu
def test_a_conversation(device_ok):
    """The operators as they are used: a prompt in two chunks of different lengths per sequence,
    two decode steps, a tree of drafts of which a path is kept, one more step.  Every step's
    attention is checked against the tokens the cache must hold by then."""
    b, hq, hkv, d, page = 3, 8, 2, 64, 16
    g = torch.Generator().manual_seed(11)
    cos, sin = b200k.rope_table(1024, d, device="cuda")
    qw, kw = ((1 + 0.1 * torch.randn(d, generator=g)).bfloat16().cuda() for _ in range(2))
    kc, vc = (torch.full((b * 16, hkv, page, d), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.randperm(b * 16, generator=g).reshape(b, 16).int().cuda()
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    kept = [[torch.empty(hkv, 0, d, dtype=torch.float64, device="cuda") for _ in range(2)] for _ in range(b)]

    def step(t, new, positions=None, mask=None):
        qkv = torch.randn(b, t, hq + 2 * hkv, d, generator=g).bfloat16().cuda()
        q, k, v = (x.transpose(1, 2) for x in qkv.split([hq, hkv, hkv], dim=2))
        n = torch.tensor(new, dtype=torch.int32, device="cuda")
        pos = lens[:, None].long() + torch.arange(t, device="cuda") if positions is None else positions
        qr = b200k.paged_kv_append(k, v, kc, vc, table, lens, cos, sin, q=q, q_weight=qw, k_weight=kw,
                                   positions=positions, new_lens=n)
        out = b200k.paged_attention(qr, kc, vc, table, lens, new_lens=n, tree_mask=mask)
        # the reference from the raw projections: one rounding of q and k on the way
        k64, q64 = (oracle.qk_rope_ref(x, w, cos, sin, pos)[0].bfloat16().double() for x, w in ((k, kw), (q, qw)))
        for i in range(b):
            if new[i] == 0:
                continue
            keys = torch.cat([kept[i][0], k64[i, :, :new[i]]], 1)
            vals = torch.cat([kept[i][1], v[i, :, :new[i]].double()], 1)
            have = kept[i][0].shape[1]
            sees = torch.ones(new[i], have + new[i], dtype=torch.bool, device="cuda")
            sees[:, have:] = (torch.ones(new[i], new[i], device="cuda").tril().bool() if mask is None
                              else mask[:new[i], :new[i]])
            for h in range(hq):
                s = q64[i, h, :new[i]] @ keys[h // 4].T / math.sqrt(d)
                p = torch.softmax(s.masked_fill(~sees, -math.inf), 1)
                want, mag = p @ vals[h // 4], p @ vals[h // 4].abs()
                # 2^-8 each for the weights and the output; and a value of q or k at a rounding
                # border may round the other way in fp32 (2^-11 of them), one step of 2^-7 in a
                # product below 4 * 4 / 8: with one such value in q and one in k a score is off
                # by 2 * 2^-6, a weight by twice that
                err = (out[i, h, :new[i]].double() - want).abs()
                assert bool((err <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -4) * mag).all())
        return k64, v

    def keep(i, k, v):
        kept[i][0] = torch.cat([kept[i][0], k], 1)
        kept[i][1] = torch.cat([kept[i][1], v.double()], 1)

    for t, new in ((33, [33, 20, 7]), (40, [5, 40, 0]), (1, [1, 1, 1]), (1, [1, 1, 1])):
        k64, v = step(t, new)
        for i in range(b):
            keep(i, k64[i, :, :new[i]], v[i, :, :new[i]])
        lens += torch.tensor(new, dtype=torch.int32, device="cuda")
    # drafts 0 - 1 - 3 and 0 - 2 - 4: the first path is accepted, its slots 0, 1 stay in place
    depth = torch.tensor([0, 1, 1, 2, 2], device="cuda")
    mask = torch.tensor([[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 1, 0, 1, 0], [1, 0, 1, 0, 1]],
                        device="cuda").bool()
    k64, v = step(5, [5, 5, 5], positions=lens[:, None] + depth, mask=mask)
    for i in range(b):
        keep(i, k64[i, :, :2], v[i, :, :2])
    lens += 2
    step(1, [1, 1, 1])                  # overwrites the slot of draft 2

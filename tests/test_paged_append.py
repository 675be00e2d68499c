"""Appending a step's keys and values to a paged cache, queries normed and rotated on the way,
against 64-bit formulas.  Values are copied: their slots, and every slot that the call does not
own, compare by their bits.  Normed and rotated rows: one rounding to their type and 32 * 2^-24 of
the magnitudes that the rotation adds up (derived in test_qk_rope.py)."""
import ctypes

import pytest
import torch

import b200k
import oracle
from b200k import _lib

EPS32 = 2.0 ** -24


class Step:
    """A step's inputs: sequences of different lengths, pages in no order, some pages unused."""

    def __init__(self, b, hq, hkv, t, d, dtype, page, lens, new=None, slots_first=False, seed=0, table=4096):
        g = torch.Generator().manual_seed(seed)
        qkv = torch.randn(b, t, hq + 2 * hkv, d, generator=g).to(dtype).cuda()
        self.q, self.k, self.v = (x.transpose(1, 2) for x in qkv.split([hq, hkv, hkv], dim=2))
        self.qw, self.kw = ((1 + 0.2 * torch.randn(d, generator=g)).to(dtype).cuda() for _ in range(2))
        self.cos, self.sin = b200k.rope_table(table, d // 16 * 16, device="cuda")
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.new = None if new is None else torch.tensor(new, dtype=torch.int32, device="cuda")
        per = max((n + t + page - 1) // page for n in lens)
        pages = b * per + 3
        self.table = torch.randperm(pages, generator=g)[:b * per].reshape(b, per).int().cuda()
        shape = (pages, page, hkv, d) if slots_first else (pages, hkv, page, d)
        self.kc, self.vc = (torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2))
        if slots_first:
            self.kc, self.vc = self.kc.transpose(1, 2), self.vc.transpose(1, 2)
        self.at = self.lens[:, None].long() + torch.arange(t, device="cuda")
        self.real = torch.ones(b, t, dtype=torch.bool, device="cuda") if new is None else (
            torch.arange(t, device="cuda") < self.new[:, None])

    def append(self, **kw):
        args = dict(q=self.q, q_weight=self.qw, k_weight=self.kw, new_lens=self.new)
        args.update(kw)
        cos, sin = (args.pop(n, getattr(self, n)) for n in ("cos", "sin"))
        return b200k.paged_kv_append(self.k, self.v, self.kc, self.vc, self.table, self.lens, cos, sin, **args)

    def check(self, before, q_out, k_weight="own", positions=None, interleaved=False, eps=1e-6, cos="own"):
        kw = self.kw if k_weight == "own" else k_weight
        c, s = (self.cos, self.sin) if cos == "own" else (None, None)
        pos = self.at if positions is None else positions
        want, scale = oracle.qk_rope_ref(self.k, kw, c, s, pos, eps, interleaved)
        args = (self.table.cpu(), self.lens.cpu(), None if self.new is None else self.new.cpu())
        kc, vc = before
        cache = oracle.paged_append_ref(want.cpu(), kc.cpu(), *args).cuda()
        mine = oracle.paged_append_ref(torch.ones_like(want).cpu(), torch.zeros_like(kc).cpu(), *args).bool().cuda()
        size = oracle.paged_append_ref(scale.cpu(), torch.zeros_like(kc).cpu(), *args).cuda()
        assert torch.equal(self.kc[~mine], kc[~mine])
        _within(self.kc, cache, size)
        assert torch.equal(self.vc, oracle.paged_append_ref(self.v.cpu(), vc.cpu(), *args).cuda())
        if q_out is not None:
            want, scale = oracle.qk_rope_ref(self.q, self.qw, c, s, pos, eps, interleaved)
            real = self.real[:, None, :, None].expand_as(want)
            _within(q_out[real], want[real], scale[real])


def _within(got, want, scale):
    u = torch.finfo(got.dtype).eps / 2
    bound = (u * want.abs() + 32 * EPS32 * scale) * (1 + u) + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"{int((err > bound).sum())} values off, worst {float((err / bound).max()):.3g} bounds"


# ---- without a GPU -----------------------------------------------------------------------------

def test_refusals_of_the_entry_point():
    h = _lib.lib()
    assert h.b200k_paged_kv_append(None, None) == _lib.INVALID_ARG

    def call(**change):
        a = _lib.PagedKvAppendArgs()
        a.batch, a.tokens, a.heads_kv, a.head_dim = 1, 4, 2, 64
        a.dtype = a.weight_dtype = _lib.BF16
        a.k = a.v = a.k_cache = a.v_cache = a.page_table = a.cache_lens = 1 << 20
        a.page_size, a.num_pages, a.max_pages, a.eps = 16, 8, 4, 1e-6
        for name, value in change.items():
            setattr(a, name, value)
        return h.b200k_paged_kv_append(ctypes.byref(a), None)

    assert call(dtype=_lib.F32) == _lib.INVALID_ARG
    assert call(page_size=0) == _lib.INVALID_ARG
    assert call(num_pages=-1) == _lib.INVALID_ARG
    assert call(head_dim=12) == _lib.UNSUPPORTED
    assert call(rotary_dim=32) == _lib.INVALID_ARG           # no table
    assert call(k_cache=None) == _lib.INVALID_ARG
    assert call(cache_lens=None) == _lib.INVALID_ARG
    assert call(q=1 << 20, heads_q=4) == _lib.INVALID_ARG    # queries without a place to go
    assert call(tokens=0, k=None) == _lib.OK


def test_refusals_of_the_wrapper():
    k = torch.zeros(1, 2, 3, 64).half()
    cache = torch.zeros(4, 2, 16, 64).half()
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        b200k.paged_kv_append(k, k, cache, cache, table, lens)
    with pytest.raises(ValueError, match="4D"):
        b200k.paged_kv_append(k, k[:, :1], cache, cache, table, lens)


# ---- on the GPU --------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("slots_first", [False, True])
@pytest.mark.parametrize("b,hq,hkv,t,d,page,lens,new", [
    (1, 4, 4, 1, 128, 16, [0], None),                             # the first token of a cache
    (3, 8, 2, 1, 128, 16, [15, 16, 17], None),                    # the last slot of a page, the first, the second
    (4, 8, 2, 5, 64, 8, [0, 3, 100, 61], [5, 1, 0, 4]),           # one sequence brings nothing
    (2, 6, 3, 70, 96, 24, [10, 1000], [70, 33]),                  # several pages a sequence
    (2, 5, 5, 9, 80, 5, [4, 22], [9, 9]),                         # pages of five tokens
    (2, 4, 1, 3, 256, 64, [62, 63], [2, 3]),
    (2, 2, 1, 4, 128, 16, [30, 7], [9, -3])])                     # counts beyond and below the step's rows
def test_append(dtype, slots_first, b, hq, hkv, t, d, page, lens, new, device_ok):
    s = Step(b, hq, hkv, t, d, dtype, page, lens, new, slots_first)
    before = s.kc.clone(), s.vc.clone()
    qo = s.append()
    assert bool((qo.transpose(1, 2)[~s.real] == 0).all())
    s.check(before, qo)


@pytest.mark.gpu
def test_rotation_norm_and_queries_are_optional(device_ok):
    for inter in (False, True):
        s = Step(2, 4, 2, 6, 64, torch.bfloat16, 16, [5, 40], [6, 2])
        before = s.kc.clone(), s.vc.clone()
        assert s.append(q=None, q_weight=None, k_weight=None, interleaved=inter) is None
        s.check(before, None, k_weight=None, interleaved=inter)
    s = Step(2, 4, 2, 6, 64, torch.bfloat16, 16, [5, 40], [6, 2])
    before = s.kc.clone(), s.vc.clone()
    s.append(q=None, q_weight=None, cos=None, sin=None)
    s.check(before, None, cos=None)
    # neither norm nor rotation: keys are copied bit for bit
    s = Step(2, 4, 2, 6, 64, torch.float16, 16, [5, 40], [6, 2])
    before = s.kc.cpu().clone()
    s.append(q=None, q_weight=None, k_weight=None, cos=None, sin=None)
    assert torch.equal(s.kc.cpu(), oracle.paged_append_ref(s.k.cpu(), before, s.table.cpu(), s.lens.cpu(), s.new.cpu()))


@pytest.mark.gpu
def test_positions_of_a_tree_and_padded_rows_stay(device_ok):
    s = Step(2, 4, 2, 6, 128, torch.bfloat16, 16, [12, 90], [6, 4])
    depth = torch.tensor([0, 1, 1, 2, 2, 3], device="cuda")
    pos = s.lens[:, None] + depth
    before = s.kc.clone(), s.vc.clone()
    q_out = torch.full((2, 4, 6, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    assert s.append(positions=pos, q_out=q_out) is q_out
    s.check(before, q_out, positions=pos)
    assert bool((q_out.transpose(1, 2)[~s.real] == 7).all())
    q_before = s.q.clone()
    s.append(positions=pos, q_out=s.q)                       # in place
    assert torch.equal(s.q.transpose(1, 2)[~s.real], q_before.transpose(1, 2)[~s.real])
    assert torch.equal(s.q.transpose(1, 2)[s.real], q_out.transpose(1, 2)[s.real])


@pytest.mark.gpu
def test_unaligned_rows_and_one_tensor_for_both_caches(device_ok):
    s = Step(2, 4, 2, 6, 64, torch.bfloat16, 16, [12, 90], [6, 4])
    s.k = torch.randn(2, 2, 6, 65, device="cuda").bfloat16()[..., 1:]
    s.v = torch.randn(2, 2, 64, 6, device="cuda").bfloat16().transpose(2, 3)
    both = torch.randn(s.kc.shape[0], 2, 2, 16, 64, device="cuda").bfloat16()
    s.kc, s.vc = both[:, 0], both[:, 1]
    before = s.kc.clone(), s.vc.clone()
    s.check(before, s.append())


@pytest.mark.gpu
def test_tokens_without_a_page_are_left_out_and_reported():
    s = Step(4, 2, 2, 3, 64, torch.float16, 16, [5, 20, 62, 14])
    s.table[0, 0] = -1                        # no page
    s.table[1, 1] = s.kc.shape[0]             # a page behind the cache
    before = s.kc.clone(), s.vc.clone()       # sequence 2: its third token lies behind the table
    s.table = s.table[:, :4]
    qo = s.append()
    s.check(before, qo)
    with pytest.raises(b200k.B200KError, match="page of sequence"):
        b200k.raise_on_device_error()
    b200k.raise_on_device_error()


@pytest.mark.gpu
def test_offsets_beyond_32_bits(device_ok):
    # two caches of 2^31 + some elements; the last pages lie behind that many elements
    page, hkv, d = 128, 8, 128
    pages = (1 << 31) // (page * hkv * d) + 4
    kc, vc = (torch.zeros(pages, hkv, page, d, dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1], [pages - 2]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([127, 3], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(2, hkv, 1, d, device="cuda").half() for _ in range(2))
    b200k.paged_kv_append(k, v, kc, vc, table, lens)
    for c, x in ((kc, k), (vc, v)):
        assert torch.equal(c[pages - 1, :, 127], x[0, :, 0]) and torch.equal(c[pages - 2, :, 3], x[1, :, 0])
        assert int(torch.count_nonzero(c[:pages - 2])) == 0 and int(torch.count_nonzero(c[pages - 2:])) <= 2 * hkv * d


@pytest.mark.gpu
def test_refused_inputs(device_ok):
    s = Step(2, 4, 2, 6, 64, torch.bfloat16, 16, [12, 90])
    call = b200k.paged_kv_append
    with pytest.raises(TypeError, match="int32"):
        call(s.k, s.v, s.kc, s.vc, s.table.long(), s.lens)
    with pytest.raises(TypeError, match="int32"):
        call(s.k, s.v, s.kc, s.vc, s.table, s.lens.long())
    with pytest.raises(ValueError, match="cache_lens must be"):
        call(s.k, s.v, s.kc, s.vc, s.table, s.lens[:1])
    with pytest.raises(ValueError, match="page_table must be"):
        call(s.k, s.v, s.kc, s.vc, s.table[:1], s.lens)
    with pytest.raises(ValueError, match="the cache holds"):
        call(s.k, s.v, s.kc[:, :1], s.vc[:, :1], s.table, s.lens)
    with pytest.raises(ValueError, match="data type"):
        call(s.k, s.v, s.kc.half(), s.vc.half(), s.table, s.lens)
    with pytest.raises(ValueError, match="contiguous rows"):
        call(s.k, s.v, s.kc[..., :1].expand(s.kc.shape), s.vc, s.table, s.lens)
    with pytest.raises(ValueError, match="come together"):
        call(s.k, s.v, s.kc, s.vc, s.table, s.lens, s.cos)
    with pytest.raises(ValueError, match="need q"):
        call(s.k, s.v, s.kc, s.vc, s.table, s.lens, q_weight=s.qw)
    with pytest.raises(ValueError, match="like k"):
        call(s.k, s.v, s.kc, s.vc, s.table, s.lens, q=s.q[:, :, :2])
    with pytest.raises(ValueError, match="device"):
        call(s.k, s.v, s.kc, s.vc, s.table.cpu(), s.lens)
    with pytest.raises(TypeError, match="float16 and bfloat16"):
        call(s.k.float(), s.v.float(), s.kc, s.vc, s.table, s.lens)


@pytest.mark.gpu
def test_captured_steps_advance(device_ok):
    # a captured step that also advances the lengths: every replay fills the next slot
    s = Step(2, 4, 2, 1, 64, torch.float16, 16, [14, 3], seed=3)
    s.append()
    torch.cuda.synchronize()
    kc0, vc0, lens0 = s.kc.clone(), s.vc.clone(), s.lens.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qo = s.append()
        s.lens += 1
    s.kc.copy_(kc0), s.vc.copy_(vc0), s.lens.copy_(lens0)
    want_k, want_v = kc0.cpu(), vc0.cpu()
    for i in range(2):
        s.k.normal_(), s.v.normal_(), s.q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        pos = (lens0 + i)[:, None]
        ref, _ = oracle.qk_rope_ref(s.k, s.kw, s.cos, s.sin, pos)
        want_k = oracle.paged_append_ref(ref.cpu(), want_k, s.table.cpu(), (lens0 + i).cpu())
        want_v = oracle.paged_append_ref(s.v.cpu(), want_v, s.table.cpu(), (lens0 + i).cpu())
        ref, scale = oracle.qk_rope_ref(s.q, s.qw, s.cos, s.sin, pos)
        _within(qo, ref, scale)
    assert torch.equal(s.lens, lens0 + 2) and torch.equal(s.vc.cpu(), want_v)
    # k: at most one rounding and 32 * 2^-24 of a sum of two magnitudes, values below 16
    assert float((s.kc.cpu().double() - want_k).abs().max()) <= 2.0 ** -11 * 16 + 32 * EPS32 * 32


@pytest.mark.gpu
def test_queries_without_key_value_heads(device_ok):
    s = Step(2, 4, 2, 6, 64, torch.bfloat16, 16, [12, 90], [6, 2])
    want = s.append()
    s.k, s.v, s.kc, s.vc = s.k[:, :0], s.v[:, :0], s.kc[:, :0], s.vc[:, :0]
    q_out = torch.full_like(want, 7.0)
    assert s.append(q_out=q_out) is q_out
    real = s.real[:, None, :, None].expand_as(want)
    assert torch.equal(q_out[real], want[real]) and bool((q_out[~real] == 7).all())
    assert torch.equal(s.append(), want)
    assert s.append(q=None, q_weight=None) is None

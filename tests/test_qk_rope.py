"""Query / key norm with rotation by position, and its gradient, against 64-bit formulas.

Tolerances: a result is rounded once to its type (half a step, u = finfo.eps / 2 relative, plus
half the smallest subnormal of float16) after a computation in fp32.  The fp32 part: the sum of
squares adds 16 products per lane and at most 4 shuffled sums (20 roundings, halved by the square
root), rsqrtf 2 ulp, five more products and sums: below 32 * 2^-24 of the magnitudes that the
rotation adds up.  The gradient of a row holds two such sums (64 * 2^-24).  A weight gradient adds,
on top, the rows of one lane group, 32 groups, the blocks in 32 strands and a shuffle: at these
sizes below 128 additions, 128 * 2^-24 of the sum of magnitudes.
"""
import ctypes
import os
import re
import shutil
import subprocess
import textwrap

import pytest
import torch

import b200k
import oracle
from b200k import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
EPS32 = 2.0 ** -24


def _within(got, want, scale, factor):
    u = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    bound = (u * want.abs() + factor * EPS32 * scale) * (1 + u) + tiny
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"{int((err > bound).sum())} values off, worst {float((err / bound).max()):.3g} bounds"


def _make(b, hq, hkv, t, d, dtype, rotary, seed=0, w_dtype=None, table=512):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(b, t, hq + 2 * hkv, d, generator=g).to(dtype).cuda()
    q, k, _ = (x.transpose(1, 2) for x in qkv.split([hq, hkv, hkv], dim=2))
    qw, kw = ((1 + 0.2 * torch.randn(d, generator=g)).to(w_dtype or dtype).cuda() for _ in range(2))
    cos, sin = b200k.rope_table(table, rotary, device="cuda")
    pos = torch.randint(0, table, (b, t), generator=g).cuda()
    return q, k, qw, kw, cos, sin, pos


def _check(q, k, qw, kw, cos, sin, pos, inter=False, **kw_args):
    got = b200k.qk_norm_rope(q, k, qw, kw, cos, sin, pos, interleaved=inter, **kw_args)
    p2 = pos if pos is not None else torch.arange(q.shape[2], device="cuda")
    p2 = p2.expand(q.shape[0], q.shape[2])
    for x, w, y in ((q, qw, got[0]), (k, kw, got[1])):
        assert y.dtype == x.dtype and y.shape == x.shape
        want, scale = oracle.qk_rope_ref(x, w, cos, sin, p2, kw_args.get("eps", 1e-6), inter)
        _within(y, want, scale, 32)
    return got


# ---- without a GPU ---------------------------------------------------------------------------

def test_refusals_of_the_entry_point():
    h = _lib.lib()
    assert h.b200k_qk_norm_rope(None, None) == _lib.INVALID_ARG
    assert h.b200k_qk_norm_rope_backward(None, None) == _lib.INVALID_ARG

    def call(**change):
        a = _lib.QkNormRopeArgs()
        a.batch, a.tokens, a.heads_q, a.heads_kv, a.head_dim, a.rotary_dim = 1, 4, 2, 2, 64, 64
        a.dtype = a.weight_dtype = _lib.BF16
        a.cos = a.sin = a.q = a.k = a.q_out = a.k_out = 1 << 20
        a.table_rows, a.table_stride, a.eps = 16, 32, 1e-6
        for name, value in change.items():
            setattr(a, name, value)
        return h.b200k_qk_norm_rope(ctypes.byref(a), None)

    assert call(tokens=-1) == _lib.INVALID_ARG
    assert call(heads_q=-1) == _lib.INVALID_ARG
    assert call(heads_kv=1 << 40) == _lib.INVALID_ARG
    assert call(head_dim=60) == _lib.UNSUPPORTED
    assert call(head_dim=264) == _lib.UNSUPPORTED
    assert call(rotary_dim=24) == _lib.UNSUPPORTED
    assert call(rotary_dim=80) == _lib.UNSUPPORTED
    assert call(dtype=_lib.E4M3) == _lib.INVALID_ARG
    assert call(weight_dtype=_lib.F16) == _lib.INVALID_ARG
    assert call(cos=None) == _lib.INVALID_ARG
    assert call(cos=(1 << 20) + 4) == _lib.UNSUPPORTED
    assert call(table_stride=31) == _lib.INVALID_ARG
    assert call(table_stride=33) == _lib.UNSUPPORTED
    assert call(eps=-1.0) == _lib.INVALID_ARG
    assert call(eps=float("nan")) == _lib.INVALID_ARG
    assert call(q=None) == _lib.INVALID_ARG
    assert call(tokens=0, q=None) == _lib.OK          # empty problems do nothing


def test_refusals_of_the_wrapper():
    q = torch.zeros(1, 2, 3, 64)
    cos, sin = b200k.rope_table(8, 64)
    with pytest.raises(ValueError, match="CUDA device"):
        b200k.qk_norm_rope(q, q, None, None, cos, sin)
    with pytest.raises(ValueError, match="4D"):
        b200k.qk_norm_rope(q[0], q, None, None, cos, sin)
    with pytest.raises(ValueError, match="agree"):
        b200k.qk_norm_rope(q, q[:, :, :2], None, None, cos, sin)
    with pytest.raises(ValueError, match="even"):
        b200k.rope_table(8, 5)


def test_table_is_taken_in_64_bits():
    cos, sin = b200k.rope_table(100001, 64, 10000.0)
    import math
    for i in (0, 1, 31):
        angle = 100000 * 10000.0 ** (-2 * i / 64)
        assert abs(float(cos[100000, i]) - math.cos(angle)) < 1e-7
        assert abs(float(sin[100000, i]) - math.sin(angle)) < 1e-7


def test_argument_structs_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    header = open(os.path.join(ROOT, "include", "b200k.h")).read()
    pairs = {"b200k_qk_norm_rope_args": _lib.QkNormRopeArgs,
             "b200k_paged_kv_append_args": _lib.PagedKvAppendArgs}
    if "b200k_paged_attention_args" in header:
        pairs["b200k_paged_attention_args"] = _lib.PagedAttentionArgs
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "b200k.h"', "int main(void) {"]
    for cname, mirror in pairs.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in mirror._fields_]
    (tmp_path / "layout.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    exe = tmp_path / "layout"
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        cname, what, value = line.split()
        mirror = pairs[cname]
        assert (ctypes.sizeof(mirror) if what == "size" else getattr(mirror, what).offset) == int(value), line
    for cname, mirror in pairs.items():   # and no field of the header is missing from the mirror
        body = re.search(r"typedef struct \{([^{}]*)\} " + cname, header).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        names = [re.sub(r"[*\s]", "", n).split(" ")[-1]
                 for decl in body.split(";") if decl.strip()
                 for n in re.sub(r"^\s*(const\s+)?\w+", "", decl.strip()).split(",")]
        assert names == [f for f, _ in mirror._fields_]


def test_oracle_gradient_against_differences():
    g = torch.Generator().manual_seed(1)
    x, dy, v = (torch.randn(2, 3, 4, 32, generator=g, dtype=torch.float64) for _ in range(3))
    w, wv = (1 + 0.3 * torch.randn(2, 32, generator=g, dtype=torch.float64)).unbind(0)
    cos, sin = b200k.rope_table(64, 16)
    pos = torch.randint(0, 64, (2, 4), generator=g)
    for inter in (False, True):
        dx, dw, _, _ = oracle.qk_rope_grad_ref(dy, x, w, cos, sin, pos, 1e-6, inter)

        def loss(step):
            return float((oracle.qk_rope_ref(x + step * v, w + step * wv, cos, sin, pos, 1e-6, inter)[0] * dy).sum())

        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        assert abs(slope - float((dx * v).sum() + (dw * wv).sum())) < 1e-6 * (1 + abs(slope))


# ---- on the GPU --------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("b,hq,hkv,t,d,rotary", [
    (1, 1, 1, 1, 128, 128),       # one row of each
    (2, 32, 8, 1, 128, 128),      # a decode step
    (2, 5, 3, 33, 64, 64),        # odd heads: the last chunk of heads is not full
    (3, 10, 5, 17, 80, 32),       # part of the head rotated
    (1, 4, 2, 7, 96, 48),         # pass-through of three vectors: the last lane holds one
    (1, 3, 1, 9, 256, 256),
    (2, 2, 1, 5, 8, 0),           # one vector, nothing to rotate
    (1, 2, 2, 3, 16, 16),
    (1, 17, 1, 130, 128, 64)])
def test_forward(dtype, inter, b, hq, hkv, t, d, rotary, device_ok):
    q, k, qw, kw, cos, sin, pos = _make(b, hq, hkv, t, d, dtype, max(rotary, 16), seed=t + d)
    if rotary == 0:
        cos, sin = (torch.empty(4, 0, device="cuda") for _ in range(2))
    _check(q, k, qw, kw, cos, sin, pos if rotary else None, inter)


@pytest.mark.gpu
def test_forward_many_rows_walks_long_chunks(device_ok):
    # enough rows that a lane group walks sixteen heads with one token's angles
    q, k, qw, kw, cos, sin, _ = _make(2, 32, 8, 2500, 128, torch.bfloat16, 128, table=2500)
    _check(q, k, qw, kw, cos, sin, None)


@pytest.mark.gpu
@pytest.mark.parametrize("w_dtype", [torch.float32, torch.bfloat16])
def test_weights_positions_and_eps(w_dtype, device_ok):
    q, k, qw, kw, cos, sin, pos = _make(3, 4, 2, 6, 128, torch.bfloat16, 128, w_dtype=w_dtype)
    _check(q, k, qw, kw, cos, sin, pos.int(), eps=1e-2)
    _check(q, k, qw, kw, cos, sin, pos[0])                                   # one row for every sequence
    _check(q, k, qw, kw, cos, sin, pos.t().contiguous().t())                 # strided positions
    _check(q, k, None, kw, cos, sin, pos)                                    # rotation alone for q
    _check(q, k, qw, kw, cos, sin, torch.full_like(pos, 511))                # the table's last row
    wide = torch.randn(512, 80, device="cuda")                               # tables with another row stride
    _check(q, k, qw, kw, wide[:, 8:72], wide[:, 3:67].contiguous(), pos)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,w_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                           (torch.float32, torch.float32)])
def test_weights_off_their_16_byte_boundaries(dtype, w_dtype, device_ok):
    for inter in (False, True):
        q, k, qw, kw, cos, sin, pos = _make(2, 3, 2, 7, 96, dtype, 32, w_dtype=w_dtype)
        odd = torch.empty(97, dtype=w_dtype, device="cuda")[1:].copy_(qw)
        _check(q, k, odd, kw, cos, sin, pos, inter)
        args = (torch.ones_like(q), torch.ones_like(k), q, k)
        got = b200k.qk_norm_rope_backward(*args, odd, kw, cos, sin, pos, interleaved=inter)
        want = b200k.qk_norm_rope_backward(*args, qw, kw, cos, sin, pos, interleaved=inter)
        assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_layouts_and_alignment(dtype, device_ok):
    q, k, qw, kw, cos, sin, pos = _make(2, 4, 2, 11, 64, dtype, 64)
    _check(q.contiguous(), k, qw, kw, cos, sin, pos)
    # rows that start one element off a 16-byte boundary, in and out
    raw = torch.randn(2, 4, 11, 65, device="cuda").to(dtype)
    odd = raw[..., 1:]
    qo = torch.zeros(2, 4, 11, 65, dtype=dtype, device="cuda")
    got = _check(odd, k, qw, kw, cos, sin, pos, q_out=qo[..., 1:])
    assert got[0].data_ptr() == qo[..., 1:].data_ptr() and bool((qo[..., 0] == 0).all())
    # a last axis that is not contiguous, a broadcast batch
    _check(torch.randn(2, 4, 64, 11, device="cuda").to(dtype).transpose(2, 3), k, qw, kw, cos, sin, pos)
    _check(q[:1].expand(2, 4, 11, 64), k, qw, kw, cos, sin, pos)
    # in place, in a fused projection
    qkv = torch.randn(2, 11, 8, 64, device="cuda").to(dtype)
    before = qkv.clone()
    views = [x.transpose(1, 2) for x in qkv.split([4, 2, 2], dim=2)]
    old = [x.transpose(1, 2) for x in before.split([4, 2, 2], dim=2)]
    b200k.qk_norm_rope(views[0], views[1], qw, kw, cos, sin, pos, q_out=views[0], k_out=views[1])
    for x, o, w in ((views[0], old[0], qw), (views[1], old[1], kw)):
        want, scale = oracle.qk_rope_ref(o, w, cos, sin, pos)
        _within(x, want, scale, 32)
    assert torch.equal(views[2], old[2])


@pytest.mark.gpu
def test_zero_rows_and_empty_calls(device_ok):
    q, k, qw, kw, cos, sin, pos = _make(2, 2, 1, 3, 64, torch.float16, 64)
    q[0] = 0
    _check(q, k, qw, kw, cos, sin, pos)
    for shape in ((0, 2, 3, 64), (2, 2, 0, 64), (2, 0, 3, 64)):
        e = torch.empty(shape, dtype=torch.float16, device="cuda")
        kk = torch.empty(shape[0], 1, shape[2], 64, dtype=torch.float16, device="cuda")
        qo, ko = b200k.qk_norm_rope(e, kk, qw, kw, cos, sin)
        assert qo.shape == e.shape and ko.shape == kk.shape
    out = b200k.qk_norm_rope_backward(torch.empty(2, 2, 0, 64, dtype=torch.float16, device="cuda"),
                                      torch.empty(2, 1, 0, 64, dtype=torch.float16, device="cuda"),
                                      q[:, :, :0], k[:, :, :0], qw, kw, cos, sin)
    assert out[0].shape == (2, 2, 0, 64) and bool((out[2] == 0).all()) and bool((out[3] == 0).all())


@pytest.mark.gpu
def test_position_outside_the_table_is_reported_and_not_read():
    q, k, qw, kw, cos, sin, pos = _make(2, 2, 1, 4, 64, torch.bfloat16, 64)
    pos[1, 2], pos[0, 0] = 512, -1
    qo, ko = b200k.qk_norm_rope(q, k, qw, kw, cos, sin, pos)
    want, scale = oracle.qk_rope_ref(q, qw, cos, sin, pos)
    assert torch.equal(torch.isnan(qo), torch.isnan(want)) and bool(torch.isnan(qo[1, :, 2]).all())
    good = ~torch.isnan(want)
    _within(qo[good], want[good], scale[good], 32)
    with pytest.raises(b200k.B200KError, match="position outside"):
        b200k.raise_on_device_error()
    b200k.raise_on_device_error()      # read once, then clear


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,w_dtype", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
                                           (torch.float32, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("b,hq,hkv,t,d,rotary", [
    (1, 1, 1, 1, 128, 128), (2, 8, 2, 37, 128, 128), (3, 10, 5, 17, 80, 32), (1, 4, 1, 50, 256, 128),
    (2, 5, 3, 9, 96, 48), (1, 8, 8, 301, 64, 64), (2, 1, 1, 3, 16, 16)])
def test_backward(dtype, w_dtype, inter, b, hq, hkv, t, d, rotary, device_ok):
    q, k, qw, kw, cos, sin, pos = _make(b, hq, hkv, t, d, dtype, rotary, seed=d + t, w_dtype=w_dtype)
    g = torch.Generator().manual_seed(9)
    dq, dk = (torch.randn(x.shape, generator=g).to(dtype).cuda() for x in (q, k))
    got = b200k.qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin, pos, interleaved=inter)
    for dy, x, w, dx, dw in ((dq, q, qw, got[0], got[2]), (dk, k, kw, got[1], got[3])):
        want_x, want_w, scale_x, scale_w = oracle.qk_rope_grad_ref(dy, x, w, cos, sin, pos, 1e-6, inter)
        assert dx.dtype == x.dtype and dw.dtype == w.dtype
        _within(dx, want_x, scale_x, 64)
        _within(dw, want_w, scale_w, 128)


@pytest.mark.gpu
def test_backward_against_differences(device_ok):
    # the slope of the 64-bit forward along a direction, against the kernel's gradients; both
    # gradients may be off by their bounds, weighed by the direction
    q, k, qw, kw, cos, sin, pos = _make(2, 3, 2, 5, 64, torch.float32, 32, seed=4)
    g = torch.Generator().manual_seed(5)
    dq, dk, vq, vk = (torch.randn(x.shape, generator=g).cuda() for x in (q, k, q, k))
    wq, wk = (torch.randn(64, generator=g).cuda() for _ in range(2))
    got = b200k.qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin, pos)
    for dy, x, w, vx, vw, dx, dw in ((dq, q, qw, vq, wq, got[0], got[2]), (dk, k, kw, vk, wk, got[1], got[3])):
        def loss(step):
            return float((oracle.qk_rope_ref(x.double() + step * vx.double(), w.double() + step * vw.double(),
                                             cos, sin, pos)[0] * dy.double()).sum())
        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        _, _, sx, sw = oracle.qk_rope_grad_ref(dy, x, w, cos, sin, pos)
        allowed = 66 * EPS32 * float((sx * vx.abs()).sum()) + 130 * EPS32 * float((sw * vw.abs()).sum()) + 1e-6 * (1 + abs(slope))
        assert abs(slope - float((dx.double() * vx).sum() + (dw.double() * vw).sum())) <= allowed


@pytest.mark.gpu
def test_backward_layouts_and_missing_weights(device_ok):
    q, k, qw, kw, cos, sin, pos = _make(2, 4, 2, 6, 64, torch.bfloat16, 64)
    one = torch.ones(1, 1, 1, 1, dtype=torch.bfloat16, device="cuda")
    dq = one.expand(q.shape)                                       # the gradient of a sum: every stride 0
    dk = torch.randn(2, 2, 6, 65, device="cuda").bfloat16()[..., 1:]   # rows off their 16-byte boundaries
    got = b200k.qk_norm_rope_backward(dq, dk, q, k, qw, None, cos, sin, pos)
    assert got[3] is None
    for dy, x, w, dx in ((dq, q, qw, got[0]), (dk, k, None, got[1])):
        want, _, scale, _ = oracle.qk_rope_grad_ref(dy, x, w, cos, sin, pos)
        _within(dx, want, scale, 64)
    again = b200k.qk_norm_rope_backward(dq, dk, q, k, qw, None, cos, sin, pos)
    assert torch.equal(again[2], got[2])                           # the same order of additions every time


@pytest.mark.gpu
def test_refused_inputs(device_ok):
    q, k, qw, kw, cos, sin, pos = _make(2, 4, 2, 6, 64, torch.bfloat16, 64)
    call = b200k.qk_norm_rope
    with pytest.raises(ValueError, match="autograd"):
        call(q, k, torch.nn.Parameter(qw), kw, cos, sin, pos)
    with torch.no_grad():
        call(q, k, torch.nn.Parameter(qw), kw, cos, sin, pos)
    with pytest.raises(ValueError, match="same data type"):
        call(q, k.half(), qw, kw, cos, sin, pos)
    with pytest.raises(TypeError):
        call(q.double(), k.double(), None, None, cos, sin, pos)
    with pytest.raises(ValueError, match="norm weights must be"):
        call(q, k, qw[:32], kw, cos, sin, pos)
    with pytest.raises(TypeError, match="one dtype"):
        call(q, k, qw.float(), kw, cos, sin, pos)
    with pytest.raises(ValueError, match="rotary_dim"):
        call(q, k, qw, kw, *b200k.rope_table(8, 128, device="cuda"), pos)
    with pytest.raises(ValueError, match="rotary_dim"):
        call(q, k, qw, kw, *b200k.rope_table(8, 40, device="cuda"), pos)
    with pytest.raises(TypeError, match="float32"):
        call(q, k, qw, kw, cos.half(), sin.half(), pos)
    with pytest.raises(TypeError, match="int32 or int64"):
        call(q, k, qw, kw, cos, sin, pos.float())
    with pytest.raises(ValueError, match="positions must be"):
        call(q, k, qw, kw, cos, sin, pos[:, :3])
    with pytest.raises(ValueError, match="device"):
        call(q, k, qw, kw, cos, sin, pos.cpu())
    with pytest.raises(ValueError, match="do not overlap"):
        call(q, k, qw, kw, cos, sin, pos, q_out=q[:1, :1, :1].expand(q.shape))
    with pytest.raises(ValueError, match="dq must have"):
        b200k.qk_norm_rope_backward(q[:1], k, q, k, qw, kw, cos, sin, pos)


@pytest.mark.gpu
def test_captured_and_on_another_stream(device_ok):
    q, k, qw, kw, cos, sin, pos = _make(2, 8, 2, 40, 128, torch.bfloat16, 128)
    dq, dk = torch.randn_like(q), torch.randn_like(k)

    def both():
        return (*b200k.qk_norm_rope(q, k, qw, kw, cos, sin, pos),
                *b200k.qk_norm_rope_backward(dq, dk, q, k, qw, kw, cos, sin, pos))

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = both()
    for _ in range(2):
        q.normal_(), dq.normal_(), pos.random_(0, 512)
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, both()):
            assert torch.equal(got, want)          # fixed order of additions: the same bits
    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:                              # two calls at once
        with torch.cuda.stream(s):
            got.append(both())
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, w) for a, w in zip(outs, want))


@pytest.mark.gpu
def test_positions_outside_the_table_name_late_tokens_as_such():
    q = torch.zeros(1, 1, 70001, 16, dtype=torch.float16, device="cuda")
    cos, sin = b200k.rope_table(70000, 16, device="cuda")
    b200k.qk_norm_rope(q, q, None, None, cos, sin)                 # token 70000: beyond the 16 bits of its place
    with pytest.raises(b200k.B200KError, match=r"token 65535 or a later one"):
        b200k.raise_on_device_error()
    b200k.qk_norm_rope(q[:, :, :65536], q[:, :, :65536], None, None, cos[:65534], sin[:65534])
    with pytest.raises(b200k.B200KError, match=r"token (65534\)|65535 or a later one)"):
        b200k.raise_on_device_error()


@pytest.mark.gpu
def test_tables_of_repeated_rows(device_ok):
    # one row for all positions through a stride of zero, one row alone
    q, k, qw, kw, cos, sin, pos = _make(2, 4, 2, 6, 64, torch.bfloat16, 64)
    _check(q, k, qw, kw, cos[7:8].expand(512, 32), sin[7:8].expand(512, 32), pos)
    _check(q, k, qw, kw, cos[7].expand(1, 32), sin[7].expand(1, 32), torch.zeros_like(pos))


@pytest.mark.gpu
def test_position_outside_the_table_leaves_what_is_not_rotated():
    q, k, qw, kw, cos, sin, pos = _make(2, 2, 1, 4, 96, torch.bfloat16, 32)
    pos[1, 2], pos[0, 0] = 512, -1
    bad = torch.zeros(2, 1, 4, 96, dtype=torch.bool, device="cuda")
    bad[1, :, 2, :32] = bad[0, :, 0, :32] = True
    for inter in (False, True):
        for x, w, y in zip((q, k), (qw, kw), b200k.qk_norm_rope(q, k, qw, kw, cos, sin, pos, interleaved=inter)):
            want, scale = oracle.qk_rope_ref(x, w, cos, sin, pos, interleaved=inter)
            assert torch.equal(torch.isnan(y), bad.expand_as(y))
            good = ~torch.isnan(want)
            _within(y[good], want[good], scale[good], 32)
        with pytest.raises(b200k.B200KError, match="position outside"):
            b200k.raise_on_device_error()
        got = b200k.qk_norm_rope_backward(q, k, q, k, qw, kw, cos, sin, pos, interleaved=inter)
        for dx, dw in (got[0::2], got[1::2]):
            rows = torch.isnan(dx)
            assert torch.equal(rows, bad.any(-1, keepdim=True).expand_as(dx))      # the mean over the row is NaN
            assert bool(torch.isnan(dw[:32]).all()) and bool(torch.isfinite(dw[32:]).all())
        with pytest.raises(b200k.B200KError, match="position outside"):
            b200k.raise_on_device_error()


def _documented_function():
    """The autograd function of README.md."""
    lines = open(os.path.join(ROOT, "README.md")).read().split("\n")
    first = lines.index("    class QkNormRope(torch.autograd.Function):")
    last = next(i for i in range(first, len(lines) + 1) if i == len(lines) or (lines[i] and not lines[i].startswith("    ")))
    scope = {"torch": torch, "b200k": b200k}
    exec(textwrap.dedent("\n".join(lines[first:last])), scope)
    return scope["QkNormRope"]


def test_the_documented_autograd_function_is_there():
    assert issubclass(_documented_function(), torch.autograd.Function)


@pytest.mark.gpu
def test_the_documented_autograd_function(device_ok):
    # a projection of queries and keys side by side, its gradient and the weights'
    function = _documented_function()
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(2, 7, 8, 64, generator=g).bfloat16().cuda().requires_grad_()
    weights = [(1 + 0.2 * torch.randn(64, generator=g)).bfloat16().cuda().requires_grad_() for _ in range(2)]
    cos, sin = b200k.rope_table(16, 32, device="cuda")
    pos = torch.randint(0, 16, (2, 7), generator=g).cuda()
    q, k, _ = (x.transpose(1, 2) for x in qkv.split([4, 2, 2], dim=2))
    qn, kn = function.apply(q, k, *weights, cos, sin, pos)
    dq, dk = (torch.randn(x.shape, generator=g).bfloat16().cuda() for x in (qn, kn))
    torch.autograd.backward((qn, kn), (dq, dk))
    first = 0
    for dy, x, w in ((dq, q, weights[0]), (dk, k, weights[1])):
        want_x, want_w, scale_x, scale_w = oracle.qk_rope_grad_ref(dy, x.detach(), w.detach(), cos, sin, pos)
        _within(qkv.grad[:, :, first:first + x.shape[1]].transpose(1, 2), want_x, scale_x, 64)
        _within(w.grad, want_w, scale_w, 128)
        first += x.shape[1]
    assert bool((qkv.grad[:, :, first:] == 0).all())
    qn, kn = function.apply(q, k, None, None, cos, sin)          # no norms, and keys that nothing uses
    dx, = torch.autograd.grad(qn.float().sum(), q)
    want, _, scale, _ = oracle.qk_rope_grad_ref(torch.ones_like(q), q.detach(), None, cos, sin,
                                                torch.arange(7, device="cuda").expand(2, 7))
    _within(dx, want, scale, 64)

"""The host module that remembers checked calls by the layouts of their tensors: what makes a new
plan and what does not, and that calls share nothing but plans."""
import ctypes
import importlib.util
import os
import shutil
import subprocess
import threading

import pytest
import torch

import b200k
from b200k import _lib, rope


def test_calls_that_cannot_have_a_plan_are_left_to_the_wrapper():
    plans = _lib.LayoutPlans("b200k_qk_norm_rope", _lib.QkNormRopeArgs)
    cpu = torch.zeros(2, 2)
    assert plans.call((cpu,), ()) is NotImplemented            # not on a GPU
    assert plans.call((None,), ("text",)) is NotImplemented    # a scalar that no kernel takes
    assert plans.call(([],), ()) is NotImplemented
    assert plans.native.size() == 0
    with pytest.raises(TypeError):
        plans.native.call((cpu,))
    with pytest.raises(ValueError, match="not a plan"):
        plans.native.add((cpu,), (), b"x" * 16, (), (), -1, 0, ())
    with pytest.raises(ValueError, match="not a plan"):        # a pointer behind the struct's end
        plans.native.add((None,), (), b"x" * 16, (), (), 12, 8, ())


def _inputs(b=2, t=5, dtype=torch.bfloat16):
    q, k = torch.randn(b, 4, t, 64, device="cuda").to(dtype), torch.randn(b, 2, t, 64, device="cuda").to(dtype)
    w = torch.ones(64, device="cuda", dtype=dtype)
    return (q, k, w, w, *b200k.rope_table(32, 64, device="cuda"))


@pytest.mark.gpu
def test_one_plan_per_layout(device_ok):
    args = _inputs()
    b200k.qk_norm_rope(*args)
    size = rope._FORWARD.native.size()
    for _ in range(3):                                          # other addresses and values
        again = _inputs()
        want = b200k.qk_norm_rope(*again)
        got = b200k.qk_norm_rope(*[x.clone() for x in again])
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    assert rope._FORWARD.native.size() == size
    b200k.qk_norm_rope(*_inputs(t=6))                           # another length
    b200k.qk_norm_rope(*args, eps=1e-3)                         # another scalar
    b200k.qk_norm_rope(*args, interleaved=True)
    b200k.qk_norm_rope(*args, q_out=torch.empty_like(args[0]))  # a given output
    with torch.no_grad():
        b200k.qk_norm_rope(*args)                               # another grad mode
    assert rope._FORWARD.native.size() == size + 5
    wide = torch.randn(2, 4, 5, 65, device="cuda").bfloat16()
    for q in (wide[..., 1:], wide[..., :64]):                   # the same strides, another alignment
        got = b200k.qk_norm_rope(q, *args[1:])[0]
        assert torch.equal(got, b200k.qk_norm_rope(q.contiguous(), *args[1:])[0])


@pytest.mark.gpu
def test_a_remembered_layout_still_refuses_gradients(device_ok):
    args = _inputs()
    b200k.qk_norm_rope(*args)
    with pytest.raises(ValueError, match="autograd"):
        b200k.qk_norm_rope(args[0].clone().requires_grad_(), *args[1:])


def test_tangents_are_refused():
    x = torch.ones(3)
    rope.check_no_grad("f", "", x, None)
    with torch.autograd.forward_ad.dual_level():
        rope.check_no_grad("f", "", x, None)
        with pytest.raises(ValueError, match="autograd"):
            rope.check_no_grad("f", "", x, torch.autograd.forward_ad.make_dual(x, x))


@pytest.mark.gpu
def test_a_remembered_layout_still_refuses_tangents(device_ok):
    args = _inputs()
    want = b200k.qk_norm_rope(*args)
    grads = b200k.qk_norm_rope_backward(*want, *args)
    cache = torch.zeros(3, 2, 16, 64, device="cuda").bfloat16()
    table, lens = (torch.zeros(shape, dtype=torch.int32, device="cuda") for shape in ((2, 1), (2,)))
    b200k.paged_kv_append(args[1], args[1], cache, cache.clone(), table, lens)
    b200k.paged_attention(args[0], cache, cache, table, lens)
    with torch.autograd.forward_ad.dual_level():
        dual = [torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)) for x in args[:2]]
        assert all(torch.equal(g, w) for g, w in zip(b200k.qk_norm_rope(*args), want))
        for call in (lambda: b200k.qk_norm_rope(args[0], dual[1], *args[2:]),
                     lambda: b200k.qk_norm_rope_backward(want[0], want[1], dual[0], *args[1:]),
                     lambda: b200k.paged_kv_append(dual[1], args[1], cache, cache.clone(), table, lens),
                     lambda: b200k.paged_attention(dual[0], cache, cache, table, lens)):
            with pytest.raises(ValueError, match="autograd"):
                call()
    again = b200k.qk_norm_rope_backward(*want, *args)
    assert all(torch.equal(g, w) for g, w in zip(again, grads))


@pytest.mark.gpu
def test_gradients_of_tables_and_outputs_are_refused(device_ok):
    q, k, w, _, cos, sin = args = _inputs()
    cache = torch.zeros(3, 2, 16, 64, device="cuda").bfloat16()
    table, lens = (torch.zeros(shape, dtype=torch.int32, device="cuda") for shape in ((2, 1), (2,)))

    def learned(x):
        return x.clone().requires_grad_()

    for call in (lambda: b200k.qk_norm_rope(q, k, w, w, learned(cos), sin),
                 lambda: b200k.qk_norm_rope(*args, q_out=learned(q)),
                 lambda: b200k.qk_norm_rope(*args, k_out=learned(k)),
                 lambda: b200k.qk_norm_rope_backward(q, k, q, k, w, w, cos, learned(sin)),
                 lambda: b200k.paged_kv_append(k, k, cache, cache.clone(), table, lens, learned(cos), sin),
                 lambda: b200k.paged_kv_append(k, k, cache, cache.clone(), table, lens, q=q, q_out=learned(q)),
                 lambda: b200k.paged_attention(q, cache, cache, table, lens, out=learned(q))):
        with pytest.raises(ValueError, match="autograd"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.gpu
def test_threads_and_streams_share_plans_only(device_ok):
    cases = [_inputs(t=5 + i % 3) for i in range(6)]
    want = [b200k.qk_norm_rope(*c) for c in cases]
    torch.cuda.synchronize()
    failed = []

    def work(number):
        with torch.cuda.stream(torch.cuda.Stream()):
            for i in range(60):
                c = (number + i) % len(cases)
                got = b200k.qk_norm_rope(*cases[c])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(g, w) for g, w in zip(got, want[c])):
                    failed.append((number, i))

    threads = [threading.Thread(target=work, args=(n,)) for n in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.gpu
def test_the_table_is_emptied_when_full(device_ok):
    args = _inputs(b=1, t=2)
    for i in range(1030):
        out = b200k.qk_norm_rope(*args, eps=1e-6 * (i + 1))
    assert rope._FORWARD.native.size() <= 1024
    assert torch.equal(out[0], b200k.qk_norm_rope(*args, eps=1e-6 * 1030)[0])


@pytest.mark.gpu
def test_a_new_layout_is_called_although_others_fill_the_table(device_ok, monkeypatch):
    # what another thread may do between a call's checks and the call
    add, args = _lib.LayoutPlans.add, _inputs(t=9)
    want = b200k.qk_norm_rope(*args, eps=1e-6)

    def add_and_fill(self, tensors, scalars, *rest, **kw):
        out = add(self, tensors, scalars, *rest, **kw)
        for i in range(1100):
            add(self, tensors, (2.0 + i, False), *rest, **kw)
        return out

    monkeypatch.setattr(_lib.LayoutPlans, "add", add_and_fill)
    args = [x.clone() for x in args]
    got = b200k.qk_norm_rope(args[0][:, :, :8], args[1][:, :, :8], *args[2:])
    assert all(torch.equal(g, w[:, :, :8]) for g, w in zip(got, want))
    assert rope._FORWARD.native.size() == 1024


@pytest.mark.gpu
def test_a_full_table_loses_one_plan_for_a_new_one(device_ok, monkeypatch):
    args, checked = _inputs(b=1, t=4), []
    check = rope._check_rows
    monkeypatch.setattr(rope, "_check_rows", lambda *a: (checked.append(1), check(*a)))
    for i in range(1100):                         # more than the table holds
        b200k.qk_norm_rope(*args, eps=1e-5 * (i + 1))
    b200k.qk_norm_rope(*args, eps=3.0)
    checked.clear()
    for i in range(100, 1100):
        b200k.qk_norm_rope(*args, eps=1e-5 * (i + 1))
    assert not checked and rope._FORWARD.native.size() == 1024
    b200k.qk_norm_rope(*args, eps=1e-5)           # the oldest has gone
    assert checked


@pytest.mark.gpu
def test_an_exception_in_an_entry_point_becomes_an_error(device_ok, tmp_path):
    # the interpreter's lock is not held in there, and is again where the error is raised
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    (tmp_path / "throws.cpp").write_text(
        '#include <stdexcept>\nextern "C" int throws(const void*, void*) { throw std::runtime_error("no room"); }\n')
    subprocess.run([cxx, "-shared", "-fPIC", "-o", tmp_path / "throws.so", tmp_path / "throws.cpp"], check=True)
    entry = ctypes.cast(ctypes.CDLL(tmp_path / "throws.so").throws, ctypes.c_void_p).value
    x = torch.ones(4, device="cuda")
    rope._FORWARD._bind()
    plans = type(rope._FORWARD.native)(entry, _lib.check)
    with pytest.raises(RuntimeError, match="no room"):
        plans.add((x,), (), b"x" * 16, ((0, 0),), ((8, 0),), -1, 0, (0,))
    for _ in range(3):
        with pytest.raises(RuntimeError, match="no room"):
            plans.call((x,), ())
    assert plans.size() == 1


def _build_module():
    spec = importlib.util.spec_from_file_location("b200k_build", os.path.join(os.path.dirname(b200k.__file__), "..", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_host_module_is_built_anew_for_another_torch_or_python(tmp_path, monkeypatch):
    build = _build_module()
    monkeypatch.setattr(build, "PLANS_STAMP", str(tmp_path / "stamp"))
    monkeypatch.setattr(build, "PLANS_PATH", str(tmp_path / "_plans.so"))
    (tmp_path / "_plans.so").write_text("")
    assert build._plans_stale("nvcc")                          # built by nobody knows what
    (tmp_path / "stamp").write_text(build._plans_stamp("nvcc"))
    assert not build._plans_stale("nvcc")
    with monkeypatch.context() as m:
        m.setattr(build.importlib.metadata, "version", lambda name: "0.0")
        assert build._plans_stale("nvcc")
    with monkeypatch.context() as m:
        m.setattr(build.sys, "version", "another")
        assert build._plans_stale("nvcc")
    assert not build._plans_stale("nvcc")
    (tmp_path / "_plans.so").unlink()
    assert build._plans_stale("nvcc")

"""The native call path of the serving-step operators (zealot_b200/calls.c) without a GPU: its tensor
checks, and that every call passes its arguments to the C function in that function's order."""
import ctypes

import numpy as np
import pytest

from test_serving_step_cpu import BOUNDS, ROPE, SCORES, SELECT, SELECTED, TABLES

CALLS = {"step_tables": TABLES, "qk_norm_rope": ROPE, "block_bounds": BOUNDS, "block_scores": SCORES,
         "select_blocks": SELECT, "paged_decode_selected": SELECTED}


def test_addresses():
    import torch
    from zealot_b200 import calls
    f, i = torch.zeros((3, 4)), torch.zeros(5, dtype=torch.int32)
    got = calls.addresses(-1, f, torch.float32, 12, None, torch.float32, 7, i, torch.int32, 5)  # -1: the CPU
    assert got == (f.data_ptr(), 0, i.data_ptr())
    assert calls.addresses(-1) == ()
    for bad in ((f, torch.float64, 12), (f, torch.float32, 11), (f.T, torch.float32, 12), (f[:, ::2], torch.float32, 6)):
        assert calls.addresses(-1, i, torch.int32, 5, *bad) == 1
    assert calls.addresses(0, f, torch.float32, 12) == 0  # another device
    assert calls.addresses(-1, torch.zeros(0), torch.float32, 0) == (0,)
    with pytest.raises(TypeError):
        calls.addresses(-1, f, torch.float32)
    with pytest.raises(TypeError):
        calls.addresses()
    with pytest.raises(AttributeError):
        calls.addresses(-1, "no tensor", torch.float32, 1)
    with pytest.raises(TypeError):
        calls.addresses(-1, f, torch.float32, "12")


def test_head_rows():
    import torch
    from zealot_b200 import calls
    f = torch.float32
    row = torch.zeros((5, 40))
    q, k = row[:, :24].unflatten(1, (6, 4)), row[:, 24:32].unflatten(1, (2, 4))
    assert calls.head_rows(-1, f, 5, 4, q, 6, k, 2) == (q.data_ptr(), 40, k.data_ptr(), 40)
    assert calls.head_rows(-1, f, 5, 4) == ()
    one = torch.zeros((5, 1, 4)).expand(5, 1, 4)
    assert calls.head_rows(-1, f, 5, 4, one, 1) == (one.data_ptr(), 4)
    for bad, heads in ((q.transpose(1, 2), 4), (q[..., ::2], 6), (q, 5), (q[:4], 6), (q.double(), 6), (row, 6), (q[None], 6)):
        assert calls.head_rows(-1, f, 5, 4, k, 2, bad, heads) == 1
    assert calls.head_rows(0, f, 5, 4, q, 6) == 0  # another device
    with pytest.raises(TypeError):
        calls.head_rows(-1, f, 5, 4, q)
    with pytest.raises(TypeError):
        calls.head_rows(-1, f, 5, "4", q, 6)
    with pytest.raises(AttributeError):
        calls.head_rows(-1, f, 5, 4, "q", 6)


def test_tensors_of_other_kinds():
    """Parameters, subclasses, views of parts, empty and single elements; types and places that no operator takes."""
    import torch
    from zealot_b200 import calls
    f = torch.float32

    class Mine(torch.Tensor):
        pass

    t = torch.zeros((4, 6))
    for x in (torch.nn.Parameter(t), t.requires_grad_(), t.as_subclass(Mine), t.detach()):
        assert calls.addresses(-1, x, f, 24) == (x.data_ptr(),)
        assert calls.addresses(-1, x, torch.bfloat16, 24) == 0
    part = t.detach()[1:3]
    assert calls.addresses(-1, part, f, 12) == (t.data_ptr() + 24,)  # an offset into its memory
    assert calls.addresses(-1, t.detach()[:, :1], f, 4) == 0
    assert calls.addresses(-1, t.detach()[:1, None, :], f, 6) == (t.data_ptr(),)  # strides of single elements do not count
    assert calls.addresses(-1, torch.zeros((0, 7)).T, f, 0) == (0,)
    assert calls.addresses(-1, torch.zeros(()), f, 1) != 0
    for kind in (torch.int32, torch.int64, torch.float32, torch.float64, torch.bfloat16, torch.float16, torch.bool):
        x = torch.zeros(3, dtype=kind)
        for other in (torch.int32, torch.int64, torch.float32, torch.float64, torch.bfloat16, torch.float16, torch.bool):
            assert calls.addresses(-1, x, other, 3) == ((x.data_ptr(),) if kind is other else 0)
    assert calls.addresses(-1, torch.zeros([1] * 8), f, 1) != 0
    with pytest.raises((TypeError, RuntimeError)):
        calls.addresses(-1, torch.zeros([1] * 9), f, 1)  # more dimensions than any argument has
    with pytest.raises((NotImplementedError, RuntimeError)):
        calls.addresses(-1, torch.zeros(3).to_sparse(), f, 3)
    assert calls.addresses(0, torch.zeros(3, device="meta"), f, 3) == 0


@pytest.mark.parametrize("name", list(CALLS))
def test_calls_pass_what_ctypes_passes(name):
    """Each argument changed in turn to one that the C function refuses in words: the same status and words."""
    from zealot_b200 import _capi, calls
    lib = _capi.load()
    base, typed, native = CALLS[name], getattr(lib, "zl_" + name), getattr(calls, name)
    pointers = {k for k, t in zip(base, _capi.SIGNATURES["zl_" + name][1]) if t is ctypes.c_void_p}
    for key in [None, *base]:
        for value in ([None] if key in pointers else [-1, 0, 7, 300, 2**30 + 1] if key else [0]):
            args = dict(base) if key is None else dict(base, **{key: value})
            args = [float(v) if k in ("eps", "scale") else v for k, v in args.items()]
            want = typed(*args), lib.zl_last_error()
            assert (native(*args), lib.zl_last_error()) == want, (key, value)


@pytest.mark.parametrize("name", list(CALLS))
def test_calls_refuse_what_does_not_fit(name):
    from zealot_b200 import calls
    args = list(CALLS[name].values())
    with pytest.raises(TypeError):
        getattr(calls, name)(*args[:-1])
    with pytest.raises(TypeError):
        getattr(calls, name)(*args, 0)
    key = "num_seqs" if "num_seqs" in CALLS[name] else "B" if "B" in CALLS[name] else "H"
    for bad, error in (("x", TypeError), (2**31, OverflowError), (2**70, OverflowError), (np.zeros(2), TypeError)):
        with pytest.raises(error):
            getattr(calls, name)(*dict(CALLS[name], **{key: bad}).values())


def test_c_floats_arrive():
    """The two float arguments, in calls that end before a device is needed."""
    from zealot_b200 import calls
    with pytest.raises(TypeError):
        calls.block_scores(*dict(SCORES, scale="x").values())
    with pytest.raises(TypeError):
        calls.qk_norm_rope(*dict(ROPE, eps=None).values())


def test_head_rows_of_none():
    import torch
    from zealot_b200 import calls
    k = torch.zeros((5, 2, 4))
    assert calls.head_rows(-1, torch.float32, 5, 4, None, 6, k, 2, None, 2) == (0, 0, k.data_ptr(), 8, 0, 0)
    assert calls.head_rows(-1, torch.float32, 5, 4, None, 6, k, 3) == 1
    with pytest.raises(TypeError):
        calls.head_rows(-1, torch.float32, 5, 4, None, None)


def test_addresses_of_shapes():
    import torch
    from zealot_b200 import calls
    f = torch.zeros((3, 4))
    assert calls.addresses(-1, f, torch.float32, (3, 4), None, torch.float32, (9,)) == (f.data_ptr(), 0)
    for bad in ((4, 3), (12,), (3, 4, 1), (1, 3, 4), (), (3, -4)):
        assert calls.addresses(-1, f, torch.float32, bad) == 0
    assert calls.addresses(-1, f.T, torch.float32, (4, 3)) == 0  # that shape, but not in order
    assert calls.addresses(-1, torch.zeros(()), torch.float32, ()) != 0
    assert calls.addresses(-1, torch.zeros((0, 7)), torch.float32, (0, 7)) == (0,)
    with pytest.raises(TypeError):
        calls.addresses(-1, f, torch.float32, (3, "4"))


@pytest.mark.parametrize("lost", ["torch.Tensor.__dlpack_c_exchange_api__ = None", "del torch.Tensor.__dlpack_c_exchange_api__"])
def test_a_torch_without_the_exchange_table(lost):
    """The tests of the checks above, with every tensor read through its methods."""
    import os
    import subprocess
    import sys
    code = f"""
import sys, torch
sys.path.insert(0, "tests")
{lost}
import test_calls_cpu as t
t.test_addresses(), t.test_head_rows(), t.test_tensors_of_other_kinds(), t.test_head_rows_of_none(), t.test_addresses_of_shapes()
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

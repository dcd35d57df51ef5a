"""PoolView is plain data: copies and pickles are views of their own, before and after a call has made the
pointer that the C entry points take."""
import copy
import ctypes
import dataclasses
import pickle

import pytest
import torch

from helm_amd.kernels import attention as ka

FIELDS = [f.name for f in dataclasses.fields(ka.PoolView)]


def made(used):
    view = ka.PoolView.of_pool(torch.randn(3, 2, 16, 64).half(), ka.alloc_v((3, 2, 16, 64), zero=True))
    if used:
        view.c_ref()
    return view


def held(ref):
    """The numbers behind a pointer that c_ref made."""
    s = ctypes.cast(ref, ctypes.POINTER(ka.KvPoolStruct)).contents
    return [getattr(s, name) for name, _ in ka.KvPoolStruct._fields_]


def numbers(view):
    return [view.k.data_ptr(), view.v.data_ptr()] + [getattr(view, x) for x in FIELDS[2:-1]]


@pytest.mark.parametrize("used", [False, True])
@pytest.mark.parametrize("make", [copy.copy, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x)),
                                  lambda x: dataclasses.replace(x)])
def test_copies(make, used):
    view = made(used)
    twin = make(view)
    assert type(twin) is ka.PoolView
    assert [getattr(twin, x) for x in FIELDS[2:]] == [getattr(view, x) for x in FIELDS[2:]]
    for x in ("k", "v"):
        assert torch.equal(getattr(twin, x), getattr(view, x))
        assert getattr(twin, x).stride() == getattr(view, x).stride()
    for x in (view, twin):                               # each has a pointer to its own numbers
        assert held(x.c_ref()) == numbers(x)


def test_a_changed_view_has_a_new_pointer():
    view = made(True)
    first = view.c_ref()
    assert view.c_ref() is first
    view.num_slots = 2
    assert held(view.c_ref()) == numbers(view) and held(view.c_ref())[-1] == 2

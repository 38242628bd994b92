"""A call with a wrong argument through the CPython entry points raises that argument's error, whatever
comes after it, and calls nothing."""

import pytest
import torch

from orchard_b200 import _lib


def names():
    _lib._load_entries()
    return [n for n in _lib._entries if n]


class Address:
    """Counts how often its address is asked for."""

    asked = 0

    def data_ptr(self):
        Address.asked += 1
        return 4096


class Whole:
    def __index__(self):
        raise OverflowError("no number")


def arguments(name, first, rest):
    sig = _lib._SIGS[name][1]
    args = [None if t is _lib._vp else 0.0 if t is _lib._f32 else 0 for t in sig]
    at = [i for i, t in enumerate(sig) if t is _lib._vp]
    args[at[0]] = first
    for i in at[1:]:
        args[i] = rest
    return args


@pytest.mark.parametrize("name", names())
def test_the_first_wrong_argument_is_the_one_reported(name):
    tensor = torch.zeros(4)
    for bad, error in ((object(), AttributeError), ("4096", AttributeError), (1.5, AttributeError)):
        with pytest.raises(error, match="data_ptr"):
            _lib._entries[name](*arguments(name, bad, tensor))
    Address.asked = 0
    with pytest.raises(AttributeError, match="data_ptr"):
        _lib._entries[name](*arguments(name, object(), Address()))
    assert Address.asked == 0  # nothing is asked of the arguments after it
    sig = _lib._SIGS[name][1]
    for t, bad, error, text in ((_lib._u32, "1", TypeError, "integer"), (_lib._u32, Whole(), OverflowError, "no number"),
                                (_lib._f32, "1", TypeError, "number|float")):
        if t not in sig:
            continue
        args = arguments(name, None, None)
        i = sig.index(t)
        args[i] = bad
        for j in range(i + 1, len(sig)):
            if sig[j] is _lib._vp:
                args[j] = tensor
        with pytest.raises(error, match=text):
            _lib._entries[name](*args)

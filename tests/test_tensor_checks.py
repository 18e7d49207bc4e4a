"""The native checks of tensors behind the Python wrappers (host/tensors.cpp)."""
import array

import pytest
import torch

HOST = -1  # the device number of host tensors


@pytest.fixture(scope="module")
def checks(tmc):
    return tmc._open_tensors()


def test_address(checks):
    x = torch.zeros(4, 6)
    assert checks.address(x, HOST, torch.float32, 24) == x.data_ptr()
    assert checks.address(x[1:], HOST, torch.float32, 18) == x.data_ptr() + 24
    assert checks.address(torch.zeros(0), HOST, torch.float32, 0) == 0


@pytest.mark.parametrize("t, device, dtype, count", [
    (torch.zeros(4), HOST, torch.float32, 5),
    (torch.zeros(4), 0, torch.float32, 1),
    (torch.zeros(4), HOST, torch.float16, 1),
    (torch.zeros(4, 4).t(), HOST, torch.float32, 1),
    (torch.zeros(8)[::2], HOST, torch.float32, 1),
    (torch.zeros(4).expand(2, 4), HOST, torch.float32, 1),
    (torch.zeros(4).to_sparse(), HOST, torch.float32, 1),
])
def test_address_refuses(checks, t, device, dtype, count):
    assert checks.address(t, device, dtype, count) is False


@pytest.mark.parametrize("args", [
    (), (torch.zeros(1),), (3, HOST, torch.float32, 1), (None, HOST, torch.float32, 1),
    (torch.zeros(1), HOST, "float32", 1), (torch.zeros(1), "0", torch.float32, 1),
    (torch.zeros(1), HOST, torch.float32, None)])
def test_address_of_other_objects(checks, args):
    with pytest.raises(TypeError):
        checks.address(*args)


def test_addresses(checks):
    pools = [torch.zeros(n, dtype=torch.float16) for n in (7, 5, 9)]
    words = array.array("Q", bytes(24))
    assert checks.addresses(pools, HOST, torch.float16, words) == 5
    assert list(words) == [t.data_ptr() for t in pools]
    assert checks.addresses(pools + pools[:0], 0, torch.float16, words) is False
    assert checks.addresses(pools, HOST, torch.float32, words) is False
    assert checks.addresses([pools[0], None], HOST, torch.float16, words) is False
    assert checks.addresses([pools[0], pools[1][::2]], HOST, torch.float16, words) is False
    for bad in ((pools * 2, HOST, torch.float16, words), (tuple(pools), HOST, torch.float16, words)):
        with pytest.raises(TypeError):
            checks.addresses(*bad)
    with pytest.raises((TypeError, BufferError)):
        checks.addresses(pools, HOST, torch.float16, bytes(24))


def sum_of_words():
    """A C function of 24 words: the sum of i times word i, as an int."""
    import ctypes as C
    kind = C.CFUNCTYPE(C.c_int, *[C.c_int64] * 24)
    return kind(lambda *w: sum(i * v for i, v in enumerate(w, 1)))


def test_call(checks):
    import ctypes as C
    f = sum_of_words()
    at = C.cast(f, C.c_void_p).value
    t = torch.zeros(4)
    assert checks.call(at, HOST) == 0
    assert checks.call(at, HOST, *range(24)) == sum(i * v for i, v in enumerate(range(24), 1))
    assert checks.call(at, HOST, 5, None, torch.int32, 3, -7) == 5 - 3 * 7
    seen = []
    g = C.CFUNCTYPE(C.c_int, C.c_int64, C.c_void_p, C.c_int64)(lambda *w: seen.append(w) or 1)
    assert checks.call(C.cast(g, C.c_void_p).value, HOST, 3, t, torch.float32, 4, 1 << 40) == 1
    assert seen == [(3, t.data_ptr(), 1 << 40)]


def test_call_refuses(checks):
    import ctypes as C
    f = sum_of_words()
    at = C.cast(f, C.c_void_p).value
    t = torch.zeros(4)
    assert checks.call(at, HOST, 1, None, torch.int32, 3, t, torch.float32, 5) == -2
    assert checks.call(at, 0, t, torch.float32, 4) == -1
    assert checks.call(at, HOST, t, torch.int32, 4) == -1
    for bad in ((), (at,), (at, HOST, 1.5), (at, HOST, t), (at, HOST, t, torch.float32),
                (at, HOST, None, 3, 4), (at, HOST, "x", torch.float32, 1), (None, HOST),
                (0, HOST), (at, HOST, *range(25)), (at, "0", 1)):
        with pytest.raises(TypeError):
            checks.call(*bad)
    with pytest.raises(OverflowError):
        checks.call(at, HOST, 1 << 70)

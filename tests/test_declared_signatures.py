"""The library's functions are declared to ctypes as in include/, and the wrappers that call
them through the native module give what is declared."""
import ctypes as C
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
KINDS = {"int64_t": C.c_int64, "int32_t": C.c_int32, "int": C.c_int32, "size_t": C.c_size_t,
         "float": C.c_float, "double": C.c_double, "uint64_t": C.c_uint64, "uint32_t": C.c_uint32}


def prototypes():
    """{name: (result, [kind of every parameter])}, pointers as c_void_p."""
    out = {}
    for header in sorted(os.listdir(os.path.join(ROOT, "include"))):
        text = open(os.path.join(ROOT, "include", header)).read()
        text = re.sub(r"/\*.*?\*/|//[^\n]*", "", text, flags=re.S)
        for result, name, params in re.findall(
                r"^((?:const\s+)?\w+\s*\**)\s*(tmc_\w+)\s*\(([^;{}]*?)\)\s*;", text, flags=re.M):
            kinds = []
            for p in re.sub(r"\s+", " ", params).split(","):
                words = [w for w in p.replace("*", " * ").replace("[", " * ").split() if w != "const"]
                if words and words != ["void"]:
                    kinds.append(C.c_void_p if "*" in words or words[0] not in KINDS
                                 else KINDS[words[0]])
            out[name] = result.replace("const", "").strip(), kinds
    return out


def plain(kind):
    """A declared kind: every pointer type as c_void_p."""
    pointer = kind in (C.c_char_p, C.c_void_p) or issubclass(kind, C._Pointer)
    return C.c_void_p if pointer else kind


DECLARED = prototypes()


def test_prototypes_are_found():
    assert len(DECLARED) > 100
    assert DECLARED["tmc_tree_layout"] == ("int", [C.c_void_p] * 4 + [C.c_int64] * 2 + [C.c_void_p])


@pytest.mark.parametrize("name", sorted(DECLARED))
def test_declared_as_in_the_header(tmc, name):
    function = getattr(tmc.lib(), name)
    if function.argtypes is None:
        pytest.skip("not declared to ctypes")
    result, kinds = DECLARED[name]
    assert [plain(k) for k in function.argtypes] == kinds
    if result in KINDS:
        assert function.restype is KINDS[result]


class Function:
    """A declared function whose call ends the test."""
    restype, address, checked = C.c_int32, 16, False

    def __init__(self, *argtypes):
        self.argtypes = list(argtypes)


T, I32 = torch.zeros(4, dtype=torch.int32), torch.int32


@pytest.mark.parametrize("takes,names,args", [
    ([C.c_void_p], "a", (T, I32, 4, 1)),                          # one too many
    ([C.c_void_p, C.c_int64, C.c_int64], "a", (T, I32, 4, 1)),    # one too few
    ([C.c_int64, C.c_void_p], "a", (T, I32, 4, 1)),               # a tensor for a number
    ([C.c_void_p, C.c_float], "a", (T, I32, 4, 1)),               # no word holds a float
    ([C.c_void_p, C.c_void_p], "a", (T, I32, 4, None, I32, 4)),   # a tensor without a name
])
def test_other_arguments_are_refused(tmc, monkeypatch, takes, names, args):
    class Module:
        @staticmethod
        def call(*_):
            raise AssertionError("called with words that are not the function's")
    monkeypatch.setattr(tmc, "_tensors", Module)
    with pytest.raises(tmc.TmcError, match="arguments"):
        tmc._call("f", -1, Function(*takes), tuple(names), *args)


def test_own_arguments_pass(tmc, monkeypatch):
    calls = []

    class Module:
        @staticmethod
        def call(*args):
            calls.append(args)
            return 0
    monkeypatch.setattr(tmc, "_tensors", Module)
    f = Function(C.c_void_p, C.c_int64, C.c_void_p, C.c_size_t, C.c_void_p, C.c_int32)
    for _ in range(2):
        tmc._call("f", -1, f, ("a", "b"), T, I32, 4, 1, None, I32, 4, 2, 3, 4)
    assert f.checked and len(calls) == 2

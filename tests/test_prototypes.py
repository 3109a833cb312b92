"""The ctypes prototypes of ``ops`` against the declarations of the C header: as many
arguments, each of the declared kind, in order; the fields of its structures too."""

import ctypes as C
import re
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

from decodebench_amd import ops  # noqa: E402

ROOT = Path(__file__).resolve().parents[1]
KINDS = {"int": C.c_int, "float": C.c_float, "unsigned": C.c_uint, "unsigned int": C.c_uint,
         "size_t": C.c_size_t, "long long": C.c_longlong}


def source():
    text = "\n".join(h.read_text() for h in sorted((ROOT / "include").glob("*.h")))
    return re.sub(r"/\*.*?\*/", "", text, flags=re.S)


def kind(declared):
    """What a declaration (with its name) is to ctypes; None for a pointer."""
    if "*" in declared:
        return None
    return KINDS[re.sub(r"\bconst\b|\w+$", "", declared.strip()).strip()]


def prototypes():
    found = re.findall(r"\b(int|size_t|const char\s*\*)\s+(db_\w+)\s*\(([^)]*)\)", source())
    return {name: (result, [] if args.strip() == "void" else args.split(","))
            for result, name, args in found}


def is_pointer(t):
    return t in (C.c_void_p, C.c_char_p) or issubclass(t, C._Pointer)


@pytest.fixture(scope="module")
def lib():
    from decodebench_amd import build

    if not ops.LIB_PATH.exists():
        build.build(verbose=False)
    return ops.load_library()


def test_the_header_is_read():
    assert len(prototypes()) >= 30
    assert kind("const void* x") is None and kind("const db_moe* m") is None
    assert kind("long long x_stride") is C.c_longlong and kind("size_t ws_bytes") is C.c_size_t


@pytest.mark.parametrize("name", sorted(prototypes()))
def test_prototype(lib, name):
    result, args = prototypes()[name]
    fn = getattr(lib, name)
    if fn.argtypes is None:
        pytest.skip("not called from Python")
    assert len(fn.argtypes) == len(args), (name, args)
    for have, declared in zip(fn.argtypes, args):
        want = kind(declared)
        assert is_pointer(have) if want is None else have is want, (name, declared, have)
    if "*" in result:
        assert fn.restype is C.c_char_p
    else:
        assert fn.restype is KINDS[result]


@pytest.mark.parametrize("name,struct", [("db_moe", ops._Moe), ("db_paged_cache", ops._PagedCache)])
def test_structure(name, struct):
    body = re.search(r"typedef struct %s \{(.*?)\}" % name, source(), flags=re.S).group(1)
    fields = []
    for line in filter(None, (s.strip() for s in body.split(";"))):
        first, *others = line.split(",")
        fields.append((re.search(r"(\w+)$", first.strip()).group(1), kind(first)))
        for other in others:
            fields.append((other.replace("*", " ").split()[-1], None if "*" in other else kind(first)))
    assert [n for n, _ in fields] == [f[0] for f in struct._fields_]
    for (field, want), (_, have) in zip(fields, struct._fields_):
        assert is_pointer(have) if want is None else have is want, field

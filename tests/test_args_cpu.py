"""The argument structs of include/nl_ops.h are the ones that
tests/test_paged_cpu.py packs by hand: a field that is added, moved or changes
its type shows here."""
import re
from pathlib import Path

import pytest

from test_paged_cpu import ARGS

HEADER = Path(__file__).resolve().parents[1] / "include" / "nl_ops.h"
SIZE = {"P": 8, "q": 8, "N": 8, "i": 4, "f": 4}


def fields(name):
    """The types of a struct's fields in order, as struct's letters."""
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    body = re.search(r"typedef struct \{([^{}]*)\} " + name + r"_args;", text).group(1)
    out = ""
    for decl in body.split(";")[:-1]:
        decl = " ".join(decl.split())
        if "*" in decl:
            assert decl.count("*") == 1 and "," not in decl
            out += "P"
        else:
            kind, letter = next((k, c) for k, c in (("long long ", "q"), ("size_t ", "N"), ("int ", "i"),
                                                    ("float ", "f")) if decl.startswith(k))
            out += letter * len(decl[len(kind):].split(","))
    return out


@pytest.mark.parametrize("name", sorted(ARGS))
def test_packed_structs(name):
    packed = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([PqNifx])", ARGS[name].format))
    have = fields(name)
    assert packed.rstrip("x") == have
    size = 0
    for c in have:                      # C's layout: each field on its own size, the whole on 8 bytes
        size = (size + SIZE[c] - 1) // SIZE[c] * SIZE[c] + SIZE[c]
    assert ARGS[name].size == (size + 7) // 8 * 8

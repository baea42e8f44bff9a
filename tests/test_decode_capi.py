"""The decode-step operators' structs are the same in the header, in the ctypes
binding and in the Rust crate: names, order, types and size (no GPU needed)."""
import ctypes as C
import os
import re

import pytest

from marian_cuda import _lib as L
from marian_cuda import build

STRUCTS = {"mc_kv4_cache": L.Kv4Cache, "mc_kv4_rows": L.Kv4Rows, "mc_kv4_attention_args": L.Kv4AttentionArgs,
           "mc_cross_attention_args": L.CrossAttentionArgs, "mc_sample_args": L.SampleArgs}
CTYPES = {"int32_t": C.c_int32, "int64_t": C.c_int64, "uint64_t": C.c_uint64, "float": C.c_float, "*": C.c_void_p}
RUST = {"int32_t": "i32", "int64_t": "i64", "uint64_t": "u64", "float": "f32"}
POINTEES = {"void": "c_void", "float": "f32", "int32_t": "i32", "uint8_t": "u8", "uint32_t": "u32"}


def header_fields(name):
    """(field, C type, pointee, const) of a struct in include/marian_cuda.h."""
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(build.REPO, "include", "marian_cuda.h")).read(), flags=re.S)
    body = re.search(r"typedef struct \{([^{}]*)\}\s*" + name + ";", text).group(1)
    fields = []
    for line in filter(None, (x.strip() for x in body.split(";"))):
        const, kind, names = re.match(r"(const )?(\w+)\s+(.*)", line, re.S).groups()
        for n in names.split(","):
            n = n.strip()
            fields.append((n.lstrip("*").strip(), "*" if n.startswith("*") else kind, kind, bool(const)))
    return fields


@pytest.mark.parametrize("name", STRUCTS)
def test_ctypes_struct_is_the_headers(name):
    want = [(f, CTYPES[kind]) for f, kind, _, _ in header_fields(name)]
    assert [tuple(x) for x in STRUCTS[name]._fields_] == want
    # every struct starts with its 8-byte members, so no padding lies between them
    sizes = [C.sizeof(t) for _, t in want]
    assert sizes == sorted(sizes, reverse=True)
    assert C.sizeof(STRUCTS[name]) == (sum(sizes) + 7) // 8 * 8


@pytest.mark.parametrize("name", STRUCTS)
def test_rust_struct_is_the_headers(name):
    text = open(os.path.join(build.ROOT, "crates", "marian-cuda", "src", "ffi.rs")).read()
    block = re.search(r"#\[repr\(C\)\]\n#\[derive\([^)]*\)\]\npub struct " + name + r" \{(.*?)\}", text, re.S).group(1)
    got = re.findall(r"pub (\w+): ([^,]+),", block)
    want = [(f, RUST[kind] if kind != "*" else f"*{'const' if const else 'mut'} {POINTEES[pointee]}")
            for f, kind, pointee, const in header_fields(name)]
    assert got == want


def test_dtypes_are_the_headers():
    text = open(os.path.join(build.REPO, "include", "marian_cuda.h")).read()
    for name, value in re.findall(r"(MC_F32|MC_F16|MC_BF16) = (\d)", text):
        assert getattr(L, name) == int(value)
        rust = open(os.path.join(build.ROOT, "crates", "marian-cuda", "src", "ffi.rs")).read()
        assert f"pub const {name}: i32 = {value};" in rust

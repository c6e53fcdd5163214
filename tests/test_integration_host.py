"""The Rust declarations of INTEGRATION.md against the library's: every function that is spelled out, parameter for parameter, and the
structs that the operators between the linears take, field for field."""
import ctypes as C
import os
import re

import pytest

from berth_b200 import _lib

with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")) as f:
    TEXT = f.read()
KINDS = {"c_int": "int", "i32": "int", "c_uint": "uint", "u32": "uint", "f32": "float", "f64": "double", "i64": "int64", "u64": "uint64", "usize": "size"}
CTYPES = {C.c_int: "int", C.c_uint: "uint", C.c_float: "float", C.c_double: "double", C.c_int64: "int64", C.c_uint64: "uint64", C.c_size_t: "size"}


def _kinds(params):
    """["int", "pointer", ..] of Rust's `name: type, ..`"""
    params = re.sub(r"/\*.*?\*/", "", params, flags=re.S)
    types = [p.split(":", 1)[1].strip() for p in params.split(",") if ":" in p]
    return ["pointer" if t.startswith("*") else KINDS[t] for t in types]


def _ctypes_kind(t):
    if t in CTYPES:     # (c_size_t and c_uint64 are one type here)
        return {"size": "uint64"}.get(CTYPES[t], CTYPES[t])
    return "pointer"


SPELLED = {m[1]: m[2] for m in re.finditer(r"pub fn (berth_\w+)\(((?:[^()]|\n)*)\)", TEXT) if "..." not in m[2]}
ROUTED = ["berth_moe_router_topk_routed", "berth_moe_layer_routed", "berth_moe_ep_send_routed", "berth_moe_p2p_send_routed"]
NEW = ["berth_ops_rope", "berth_ops_rope_frequencies", "berth_ops_logprobs", "berth_moe_route"] + ROUTED


@pytest.mark.parametrize("name", sorted(set(SPELLED) & set(_lib.SIGNATURES) | set(NEW)))
def test_a_declared_function_is_the_library_s(name):
    assert name in SPELLED, f"INTEGRATION.md does not spell out {name}"
    want = [_ctypes_kind(t) for t in _lib.SIGNATURES[name][1]]
    assert [{"size": "uint64"}.get(k, k) for k in _kinds(SPELLED[name])] == want


@pytest.mark.parametrize("name,struct", [("BerthMoeRouting", _lib.MoeRouting), ("BerthRopeRows", _lib.RopeRows), ("BerthRopeScaling", _lib.RopeScaling)])
def test_a_declared_struct_is_the_library_s(name, struct):
    m = re.search(r"#\[repr\(C\)\] pub struct " + name + r" \{(.*?)\}", TEXT, re.S)
    assert m, f"INTEGRATION.md does not define {name}"
    body = re.sub(r"/\*.*?\*/", "", m[1], flags=re.S)
    fields = [p.split(":")[0].replace("pub ", "").strip() for p in body.split(",") if ":" in p]
    assert fields == [n for n, _ in struct._fields_]
    assert _kinds(body) == [_ctypes_kind(t) for _, t in struct._fields_]


def test_every_struct_that_these_declarations_name_is_defined():
    for name in set(re.findall(r"\*(?:const|mut) (Berth(?:Rope|Moe)\w+)", TEXT)):
        assert re.search(r"pub struct " + name + r"\b", TEXT), name

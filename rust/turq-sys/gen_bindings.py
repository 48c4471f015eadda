"""Writes src/lib.rs of the `turq-sys` crate from include/turq.h, and is the parser the
signature-drift test uses (tests/test_rust_binding.py). Run from the repository root:

    python rust/turq-sys/gen_bindings.py

Only the constructs turq.h uses are understood: `#define NAME value` constants, the two enums,
opaque structs and plain function declarations with pointer / integer / float parameters."""
from __future__ import annotations

import os
import re

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(HERE, "..", "..", "include", "turq.h")
OUT = os.path.join(HERE, "src", "lib.rs")

SCALARS = {"int32_t": "i32", "int64_t": "i64", "size_t": "usize", "float": "f32", "double": "f64", "char": "c_char", "void": "c_void",
           "turq_ctx": "turq_ctx", "turq_qtensor": "turq_qtensor", "turq_tp": "turq_tp",
           "turq_host_call": "turq_host_call", "turq_kv_cache": "turq_kv_cache"}


def strip_comments(text: str) -> str:
    return re.sub(r"/\*.*?\*/", " ", text, flags=re.S)


def c_type_to_rust(ctype: str) -> str:
    """`const turq_qtensor* const*` -> `*const *const turq_qtensor`; a bare scalar -> its Rust name."""
    toks = re.findall(r"const|\*|[A-Za-z_][A-Za-z_0-9]*", ctype)
    base, const_base = None, False
    i = 0
    while i < len(toks) and toks[i] != "*":
        if toks[i] == "const":
            const_base = True
        else:
            base = toks[i]
        i += 1
    if base not in SCALARS:
        raise ValueError(f"unknown C type {ctype!r}")
    rust = SCALARS[base]
    pointee_const = const_base
    while i < len(toks):
        assert toks[i] == "*"
        i += 1
        next_const = False
        while i < len(toks) and toks[i] == "const":
            next_const = True
            i += 1
        rust = ("*const " if pointee_const else "*mut ") + rust
        pointee_const = next_const
    return rust


def parse_header(path: str = HEADER):
    """Returns (functions, constants, enums): functions = [(name, rust return type, [(arg, rust type)])]."""
    text = strip_comments(open(path).read())
    consts = [(m.group(1), m.group(2).strip()) for m in re.finditer(r"#define\s+(TURQ_[A-Z_0-9]+)\s+(.+)", text)
              if m.group(1) != "TURQ_H"]
    enums = []
    for m in re.finditer(r"typedef\s+enum\s*\{(.*?)\}\s*(\w+)\s*;", text, flags=re.S):
        items = [(a.strip(), int(b)) for a, b in re.findall(r"(\w+)\s*=\s*(-?\d+)", m.group(1))]
        enums.append((m.group(2), items))
    body = re.sub(r"typedef\s+enum\s*\{.*?\}\s*\w+\s*;", " ", text, flags=re.S)
    body = re.sub(r"typedef\s+struct\s+\w+\s+\w+\s*;", " ", body)
    body = re.sub(r"#.*", " ", body)
    body = body.replace('extern "C" {', " ").replace("}", " ")
    funcs = []
    for m in re.finditer(r"([A-Za-z_][\w\s\*]*?)\b(turq_\w+)\s*\(([^;{]*?)\)\s*;", body, flags=re.S):
        ret, name, args = m.group(1).strip(), m.group(2), m.group(3).strip()
        rargs = []
        if args and args != "void":
            for a in args.split(","):
                a = " ".join(a.split())
                am = re.match(r"(.*?)([A-Za-z_]\w*)$", a)
                rargs.append((am.group(2), c_type_to_rust(am.group(1))))
        rret = c_type_to_rust(ret)
        funcs.append((name, rret, rargs))
    return funcs, consts, enums


def parse_rust(path: str = OUT):
    """The extern block of lib.rs -> [(name, return type, [(arg, type)])]."""
    text = re.sub(r"//.*", "", open(path).read())
    block = re.search(r'extern\s+"C"\s*\{(.*)\}', text, flags=re.S).group(1)
    funcs = []
    for m in re.finditer(r"pub\s+fn\s+(\w+)\s*\((.*?)\)\s*(?:->\s*([^;]+?))?\s*;", block, flags=re.S):
        args = []
        for a in filter(None, (s.strip() for s in m.group(2).split(","))):
            an, at = a.split(":", 1)
            args.append((an.strip(), " ".join(at.split())))
        funcs.append((m.group(1), " ".join((m.group(3) or "()").split()), args))
    return funcs


def render() -> str:
    funcs, consts, enums = parse_header()
    out = ["//! Raw bindings to `libturq.so` (include/turq.h). Generated by gen_bindings.py; do not edit.",
           "//!",
           "//! Every entry returns a `turq_status` as `i32` (0 = OK) and never unwinds across the boundary.",
           "#![allow(non_camel_case_types)]",
           "#![no_std]",
           "",
           "use core::ffi::{c_char, c_void};",
           ""]
    for name in ("turq_ctx", "turq_qtensor", "turq_tp", "turq_host_call", "turq_kv_cache"):
        out += [f"/// Opaque handle owned by the library.", "#[repr(C)]", f"pub struct {name} {{", "    _private: [u8; 0],", "}", ""]
    for name, value in consts:
        value = value.replace("(4 << 20)", "4 << 20")
        ty = "usize" if "BYTES" in name else "i32"
        out.append(f"pub const {name}: {ty} = {value};")
    out.append("")
    for ename, items in enums:
        out.append(f"// enum {ename}")
        for iname, ival in items:
            out.append(f"pub const {iname}: i32 = {ival};")
        out.append("")
    out.append('extern "C" {')
    for name, ret, args in funcs:
        arglist = ", ".join(f"{a}: {t}" for a, t in args)
        line = f"    pub fn {name}({arglist})" + ("" if ret == "c_void" else f" -> {ret}") + ";"
        if len(line) > 110:
            inner = ",\n".join(f"        {a}: {t}" for a, t in args)
            line = f"    pub fn {name}(\n{inner},\n    )" + ("" if ret == "c_void" else f" -> {ret}") + ";"
        out.append(line)
    out.append("}")
    return "\n".join(out) + "\n"


if __name__ == "__main__":
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    with open(OUT, "w") as f:
        f.write(render())
    print(OUT)

#!/usr/bin/env python
"""Writes src/lib.rs: the Rust `extern "C"` declarations of every TQ_API entry point of include/tangq.h.

tang is a Rust workspace; this crate is what tang-compute / tang-infer would depend on to reach libtangq.
No Rust toolchain exists where this library is developed, so the crate is source only: the declarations are
generated from the header (this script), and tests/test_rust_binding.py checks that the committed src/lib.rs
is what the generator produces from the current header and that it declares every exported symbol.

    python rust/tangq-sys/gen_bindings.py            # rewrite src/lib.rs
"""
from __future__ import annotations

import os
import re

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(HERE, "..", "..", "include", "tangq.h")

SCALARS = {
    "int": "c_int", "size_t": "usize", "float": "f32", "double": "f64", "uint32_t": "u32", "uint64_t": "u64",
    "int8_t": "i8", "unsigned long long": "u64", "unsigned": "c_uint", "char": "c_char", "void": "c_void",
}
OPAQUE = re.findall(r"typedef struct (tq_\w+) \1;", open(HEADER).read())     # handles: pointers to them is all that a caller has


def strip_comments(text: str) -> str:
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return "\n".join(l for l in text.split("\n") if not l.lstrip().startswith("#"))   # preprocessor lines


def rust_type(ctype: str) -> str:
    """C parameter / return type (without the name) -> Rust."""
    t = " ".join(ctype.replace("*", " * ").split())
    if t == "void":
        return "()"
    stars = t.count("*")
    base = t.replace("*", " ").replace("const", " ")
    base = " ".join(base.split())
    if base in SCALARS:
        rt = SCALARS[base]
    elif base in OPAQUE or base.startswith("tq_"):
        rt = base
    else:
        raise ValueError(f"unknown C type {ctype!r}")
    if stars == 0:
        return rt
    # constness of each pointer level, outermost last: "const T* const*" -> [const, const]
    parts = [p.strip() for p in t.split("*")]
    quals = []
    for i in range(stars):
        seg = parts[i] if i == 0 else parts[i]
        quals.append("const" in seg.split())
    out = rt
    for is_const in quals:
        out = f"*const {out}" if is_const else f"*mut {out}"
    return out


def split_param(p: str):
    p = " ".join(p.split())
    m = re.match(r"^(.*?)([A-Za-z_][A-Za-z0-9_]*)$", p)
    ctype, name = m.group(1).strip(), m.group(2)
    if name in ("type", "ref", "move", "in", "fn"):
        name += "_"
    return ctype, name


def parse(text: str):
    text = strip_comments(text)
    structs = []
    for m in re.finditer(r"typedef struct (tq_\w+) \{(.*?)\} \1;", text, flags=re.S):
        fields = []
        for decl in m.group(2).split(";"):
            decl = " ".join(decl.split())
            if not decl:
                continue
            ctype, first = split_param(decl.split(",")[0])
            names = [first] + [n.strip() for n in decl.split(",")[1:]]
            fields += [(n, rust_type(ctype)) for n in names]
        structs.append((m.group(1), fields))
    funcs = []
    for m in re.finditer(r"TQ_API\s+([A-Za-z_][A-Za-z0-9_ \*]*?)\s*\b(tq_\w+)\s*\(([^;]*?)\)\s*;", text, flags=re.S):
        ret, name, params = " ".join(m.group(1).split()), m.group(2), m.group(3)
        plist = []
        if params.strip() not in ("", "void"):
            for p in params.split(","):
                ctype, pname = split_param(p)
                plist.append((pname, rust_type(ctype)))
        funcs.append((name, rust_type(ret), plist))
    enums = {}
    for m in re.finditer(r"typedef enum (tq_\w+) \{(.*?)\} \1;", text, flags=re.S):
        items = []
        for it in m.group(2).split(","):
            it = " ".join(it.split())
            if it:
                k, v = [x.strip() for x in it.split("=")]
                items.append((k, int(v)))
        enums[m.group(1)] = items
    return structs, funcs, enums


def render(structs, funcs, enums) -> str:
    out = ["//! Raw bindings to libtangq (generated by gen_bindings.py from include/tangq.h; do not edit).",
           "#![allow(non_camel_case_types)]", "",
           "use std::os::raw::{c_char, c_int, c_uint, c_void};", ""]
    for name in OPAQUE:
        out += ["#[repr(C)]", f"pub struct {name} {{", "    _private: [u8; 0],", "}", ""]
    for ename, items in enums.items():
        for k, v in items:
            out.append(f"pub const {k}: c_int = {v};")
        out.append("")
    for name, fields in structs:
        out += ["#[repr(C)]", "#[derive(Clone, Copy, Debug)]", f"pub struct {name} {{"]
        out += [f"    pub {n}: {t}," for n, t in fields]
        out += ["}", ""]
    out.append('#[link(name = "tangq")]')
    out.append('extern "C" {')
    for name, ret, params in funcs:
        args = ", ".join(f"{n}: {t}" for n, t in params)
        out.append(f"    pub fn {name}({args})" + ("" if ret == "()" else f" -> {ret}") + ";")
    out += ["}", ""]
    return "\n".join(out)


def generate() -> str:
    return render(*parse(open(HEADER).read()))


if __name__ == "__main__":
    path = os.path.join(HERE, "src", "lib.rs")
    with open(path, "w") as f:
        f.write(generate())
    print("wrote", path)

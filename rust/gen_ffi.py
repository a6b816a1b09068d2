#!/usr/bin/env python
"""Generates rust/src/ffi.rs (the `extern "C"` block of the shim crate) from include/lumen_b200.h.

    python rust/gen_ffi.py            # rewrite rust/src/ffi.rs
    python rust/gen_ffi.py --check    # exit 1 if the committed file is out of date

One Rust declaration per C declaration, in header order, so that the shim can never bind a function the library
does not export or miss one it does.  tests/test_rust_shim.py runs the check and compares the names with the
symbols the built library exports.
"""
from __future__ import annotations

import re
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "lumen_b200.h"
OUT = ROOT / "rust" / "src" / "ffi.rs"

OPAQUE = ["lumen_ctx", "lumen_tensor", "lumen_rope", "lumen_kv_cache", "lumen_llama_kv_cache", "lumen_self_attention",
          "lumen_llama", "lumen_model", "lumen_page_pool", "lumen_page_batch"]
STRUCTS = ["lumen_llama_config", "lumen_decoder_layer", "lumen_decoder_config", "lumen_sample_params"]
SCALARS = {"int": "c_int", "float": "f32", "double": "f64", "size_t": "usize", "uint64_t": "u64", "int64_t": "i64", "int32_t": "i32",
           "uint16_t": "u16", "char": "c_char", "void": "c_void", "lumen_dtype": "c_int"}


def strip_comments(text: str) -> str:
    return re.sub(r"/\*.*?\*/", " ", text, flags=re.S)


def c_functions(text: str):
    """(return type, name, [(type, name)]) for every function declared in the header."""
    text = strip_comments(text)
    out = []
    for m in re.finditer(r"^([A-Za-z_][A-Za-z0-9_ \*]*?)\b(lumen_[a-z0-9_]+)\s*\(([^;{]*?)\)\s*;", text, flags=re.M | re.S):
        ret, name, args = m.group(1).strip(), m.group(2), " ".join(m.group(3).split())
        params = []
        if args and args != "void":
            for a in args.split(","):
                a = a.strip()
                arr = re.match(r"(.*?)(\w+)\s*\[\d*\]$", a)  # `size_t out[6]` decays to a pointer
                if arr:
                    params.append((arr.group(1).strip() + " *", arr.group(2)))
                    continue
                pm = re.match(r"(.*?)(\w+)$", a)
                params.append((pm.group(1).strip(), pm.group(2)))
        out.append((ret, name, params))
    return out


def rust_type(c: str) -> str:
    """`const void *const *` -> `*const *const c_void`: a pointer is `*const` when what it points at is const."""
    parts = [" ".join(p.split()) for p in c.split("*")]
    base_tokens = parts[0].split()
    pointee_const = "const" in base_tokens
    base = " ".join(t for t in base_tokens if t != "const")
    t = base if (base in OPAQUE or base in STRUCTS) else SCALARS[base]
    for qual in parts[1:]:  # one entry per '*', holding the qualifiers written after it
        t = ("*const " if pointee_const else "*mut ") + t
        pointee_const = "const" in qual.split()
    return t


def c_struct(text: str, name: str):
    m = re.search(r"typedef struct \{([^{}]*)\}\s*" + name + r"\s*;", strip_comments(text))
    fields = []
    for line in m.group(1).split(";"):
        line = " ".join(line.split())
        if line:
            pm = re.match(r"(.*?)(\w+)$", line)
            fields.append((pm.group(1).strip(), pm.group(2)))
    return fields


def generate() -> str:
    text = HEADER.read_text()
    lines = ["// GENERATED by rust/gen_ffi.py from include/lumen_b200.h - do not edit by hand.",
             "// Raw bindings of liblumen_b200.so.  Not compiled or tested where this was written (no rustc).",
             "#![allow(non_camel_case_types)]", "",
             "use std::os::raw::{c_char, c_int, c_void};", ""]
    for code, val in re.findall(r"#define (LUMEN_(?:OK|ERR_[A-Z_]+|W_[QKVO]|MLP_[A-Z]+|NCCL_ID_BYTES)) (\d+)", text):
        lines.append(f"pub const {code}: c_int = {val};")
    lines += ["pub const LUMEN_F32: c_int = 0;", "pub const LUMEN_BF16: c_int = 1;", ""]
    for o in OPAQUE:
        lines += ["#[repr(C)]", f"pub struct {o} {{", "    _private: [u8; 0],", "}"]
    for s in STRUCTS:
        lines += ["", "#[repr(C)]", "#[derive(Clone, Copy, Debug)]", f"pub struct {s} {{"]
        for ty, nm in c_struct(text, s):
            lines.append(f"    pub {nm}: {rust_type(ty)},")
        lines.append("}")
    lines += ["", '#[link(name = "lumen_b200")]', 'extern "C" {']
    for ret, name, params in c_functions(text):
        args = ", ".join(f"{nm}: {rust_type(ty)}" for ty, nm in params)
        r = "" if ret == "void" else f" -> {rust_type(ret)}"
        lines.append(f"    pub fn {name}({args}){r};")
    lines += ["}", ""]
    return "\n".join(lines)


if __name__ == "__main__":
    new = generate()
    if "--check" in sys.argv:
        sys.exit(0 if OUT.exists() and OUT.read_text() == new else 1)
    OUT.write_text(new)
    print(f"wrote {OUT} ({len(c_functions(HEADER.read_text()))} functions)")

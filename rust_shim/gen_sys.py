"""Generates rust_shim/src/cuda/sys.rs: the `extern "C"` block a Rust crate binds libnrs_b200.so with, one
declaration per entry point of include/*.h (parsed, not hand-kept).  Run: python rust_shim/gen_sys.py"""
from __future__ import annotations

import re
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))

SCALARS = {"int": "i32", "float": "f32", "double": "f64", "size_t": "usize", "int64_t": "i64", "uint64_t": "u64",
           "int32_t": "i32", "char": "c_char", "void": "c_void"}
OPAQUE = ["nrs_ctx", "nrs_node", "nrs_adamw", "nrs_trainer", "nrs_dp", "nrs_checkpoint"]
STRUCTS = ["nrs_layer_spec", "nrs_named_tensor"]
RUST_KEYWORDS = {"type", "ref", "in", "fn", "mod", "move", "box", "loop", "match", "self", "use", "where", "impl"}

HEADER = '''// GENERATED by rust_shim/gen_sys.py from include/nrs.h, nrs_graph.h, nrs_checkpoint.h — do not edit.
// Raw bindings of libnrs_b200.so for the `neuralrs` crate (module `cuda::sys`).
#![allow(non_camel_case_types, dead_code)]
use std::os::raw::{c_char, c_void};

macro_rules! opaque { ($($n:ident),*) => { $( #[repr(C)] pub struct $n { _private: [u8; 0] } )* } }
opaque!(%s);

/// nrs_layer_spec (nrs_graph.h): one layer of the native trainer's model description.
#[repr(C)]
#[derive(Clone, Copy, Debug, Default)]
pub struct nrs_layer_spec { pub kind: i32, pub a: i32, pub b: i32, pub c: i32, pub d: i32, pub e: i32 }

/// nrs_named_tensor (nrs_checkpoint.h): NamedTensor of src/serialize.rs:160.
#[repr(C)]
pub struct nrs_named_tensor { pub name: *const c_char, pub shape: *const i64, pub ndim: i32, pub data: *const f32 }

/// Poll function of nrs_watchdog_wait: 0 = still running, 1 = finished, negative = failed.
pub type nrs_poll_fn = Option<unsafe extern "C" fn(user: *mut c_void) -> i32>;

pub const NRS_OK: i32 = 0;
pub const NRS_ERR_ARG: i32 = 1;
pub const NRS_ERR_SHAPE: i32 = 2;
pub const NRS_ERR_ALLOC: i32 = 3;
pub const NRS_ERR_CUDA: i32 = 4;
pub const NRS_ERR_NCCL: i32 = 5;
pub const NRS_ERR_TIMEOUT: i32 = 6;
pub const NRS_ERR_UNSUPPORTED: i32 = 7;
pub const NRS_MATH_3XTF32: i32 = 0;
pub const NRS_MATH_TF32: i32 = 1;
pub const NRS_MATH_FP32: i32 = 2;
pub const NRS_ACT_NONE: i32 = 0;
pub const NRS_ACT_RELU: i32 = 1;
pub const NRS_ACT_GELU: i32 = 2;
pub const NRS_ACT_SILU: i32 = 3;

extern "C" {
'''


def rust_type(decl: str) -> str:
    """Rust spelling of a C type written without a parameter name."""
    d = decl.strip()
    if d == "nrs_poll_fn":
        return "nrs_poll_fn"
    # peel pointers from the right: each '*' may be preceded by a const that applies to the pointee
    m = re.match(r"^(.*?)(\*\s*(const)?\s*)$", d)
    if m:
        inner = m.group(1).strip()
        # `T* const` (a const pointer) qualifies the pointer itself, which Rust does not spell
        pointee_const = inner.startswith("const ") or inner.endswith(" const")
        inner_clean = re.sub(r"^const\s+|\s+const$", "", inner).strip() if not inner.rstrip().endswith("*") else inner
        if inner.rstrip().endswith("*") or inner.rstrip().endswith("* const"):
            # pointer to pointer: constness of the outer pointee is that of the inner pointer
            outer_const = inner.rstrip().endswith("const")
            inner_ptr = inner[: -len("const")].strip() if outer_const else inner
            return ("*const " if outer_const else "*mut ") + rust_type(inner_ptr)
        return ("*const " if pointee_const else "*mut ") + rust_type(inner_clean)
    base = re.sub(r"\bconst\b", "", d).strip()
    if base in SCALARS:
        return SCALARS[base]
    if base in OPAQUE or base in STRUCTS:
        return base
    raise ValueError(f"no Rust spelling for C type `{decl}`")


def split_param(p: str) -> tuple[str, str]:
    m = re.match(r"^(.*?)(\w+)$", p.strip(), flags=re.S)
    ctype, name = m.group(1).strip(), m.group(2)
    if name in RUST_KEYWORDS:
        name += "_"
    return ctype, name


def generate() -> str:
    from neuralrs_b200 import _lib
    out = [HEADER % ", ".join(OPAQUE)]
    for name, (ret, params) in sorted(_lib.declared_functions().items()):
        args = []
        for p in params:
            ctype, pname = split_param(p)
            args.append(f"{pname}: {rust_type(ctype)}")
        r = "" if ret.strip() == "void" else f" -> {rust_type(ret)}"
        out.append(f"    pub fn {name}({', '.join(args)}){r};\n")
    out.append("}\n")
    return "".join(out)


if __name__ == "__main__":
    dst = Path(__file__).resolve().parent / "src" / "cuda" / "sys.rs"
    dst.write_text(generate())
    print(dst)

"""Generates engine-mlx_b200/rust/engine-mlx-ffi/src/sys.rs — the raw Rust
declarations of include/emx.h (constants, opaque handles, callback types,
#[repr(C)] structs and one extern "C" fn per header prototype) — so the crate
that replaces crates/mlx-ffi binds exactly the header's ABI.

    python engine-mlx_b200/rust/gen_sys.py [--check]

--check exits non-zero when sys.rs differs from what the header gives (the
CPU test-suite runs it)."""
import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(HERE, "..", "..", "include", "emx.h")
OUT = os.path.join(HERE, "engine-mlx-ffi", "src", "sys.rs")

SCALAR = {"int": "c_int", "float": "f32", "int32_t": "i32", "int64_t": "i64", "uint64_t": "u64",
          "size_t": "usize", "char": "c_char", "void": "c_void", "emx_dtype": "c_int",
          "emx_error_handler": "emx_error_handler", "emx_token_cb": "emx_token_cb"}
OPAQUE = ["emx_ctx", "emx_comm", "emx_qwen3"]
STRUCTS = ["emx_qwen3_config", "emx_st_tensor", "emx_paged_kv", "emx_paged_batch"]
RUST_KEYWORDS = {"type", "ref", "mut", "fn", "in", "loop", "match", "move", "self", "use", "where"}


def rust_type(ct):
    ct = ct.strip()
    stars = ct.count("*")
    base = ct.replace("*", "").strip()
    const = base.startswith("const ")
    base = base.replace("const ", "").strip()
    if base in SCALAR:
        rt = SCALAR[base]
    elif base in OPAQUE or base in STRUCTS:
        rt = base
    else:
        raise ValueError(f"unmapped C type {ct!r}")
    for i in range(stars):
        rt = ("*const " if (const and i == 0) else "*mut ") + rt
    return rt


def parse(header):
    src = open(header).read()
    nocomment = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    consts = re.findall(r"^#define\s+(EMX_[A-Z0-9_]+)\s+(-?\d+)", nocomment, flags=re.M)
    enums = re.findall(r"typedef enum\s*\{([^}]*)\}\s*(\w+)\s*;", nocomment)
    structs = {}
    for body, name in re.findall(r"typedef struct\s*\{(.*?)\}\s*(\w+)\s*;", nocomment, flags=re.S):
        fields = []
        for decl in body.split(";"):
            decl = " ".join(decl.split())
            if not decl:
                continue
            m = re.match(r"^((?:const\s+)?[\w]+\s*\**)\s*(.*)$", decl)
            ty, names = m.group(1).strip(), m.group(2)
            for n in names.split(","):
                n = n.strip()
                am = re.match(r"^(\w+)\[(\d+)\]$", n)
                if am:
                    fields.append((am.group(1), f"[{rust_type(ty)}; {am.group(2)}]"))
                else:
                    fields.append((n, rust_type(ty)))
        structs[name] = fields
    protos = []
    for ret, name, args in re.findall(r"^\s*((?:const\s+)?[\w]+\s*\**)\s*(emx_\w+)\s*\(([^;{]*?)\)\s*;", nocomment,
                                      flags=re.M):
        params = []
        for a in args.split(","):
            a = " ".join(a.split())
            if not a or a == "void":
                continue
            m = re.match(r"^(.*?)(\w+)\s*$", a)
            ty, pname = m.group(1).strip(), m.group(2)
            if pname in RUST_KEYWORDS:
                pname = pname + "_"
            params.append((pname, rust_type(ty)))
        r = ret.strip()
        protos.append((name, params, None if r == "void" else rust_type(r)))
    return consts, enums, structs, protos


def render(header):
    consts, enums, structs, protos = parse(header)
    o = ["// @generated by engine-mlx_b200/rust/gen_sys.py from include/emx.h -- do not edit.",
         "#![allow(non_camel_case_types, non_snake_case, dead_code)]", "",
         "use std::os::raw::{c_char, c_int, c_void};", ""]
    for n, v in consts:
        o.append(f"pub const {n}: c_int = {v};")
    o.append("")
    for body, _name in enums:
        for item in body.split(","):
            item = item.strip()
            if item:
                k, v = [x.strip() for x in item.split("=")]
                o.append(f"pub const {k}: c_int = {v};")
    o.append("")
    for t in OPAQUE:
        o += ["#[repr(C)]", f"pub struct {t} {{", "    _private: [u8; 0],", "}"]
    o.append("")
    o.append("pub type emx_error_handler = Option<unsafe extern \"C\" fn(msg: *const c_char, data: *mut c_void)>;")
    o.append("pub type emx_token_cb = Option<unsafe extern \"C\" fn(token: i32, index: c_int, user: *mut c_void) "
             "-> c_int>;")
    o.append("")
    for name in STRUCTS:
        o += ["#[repr(C)]", "#[derive(Clone, Copy)]", f"pub struct {name} {{"]
        for f, t in structs[name]:
            o.append(f"    pub {f}: {t},")
        o += ["}", ""]
    o.append("extern \"C\" {")
    for name, params, ret in protos:
        ps = ", ".join(f"{p}: {t}" for p, t in params)
        o.append(f"    pub fn {name}({ps})" + (f" -> {ret};" if ret else ";"))
    o.append("}")
    return "\n".join(o) + "\n", [p[0] for p in protos]


def main():
    text, names = render(HEADER)
    if "--check" in sys.argv:
        cur = open(OUT).read() if os.path.exists(OUT) else ""
        if cur != text:
            print("sys.rs is out of date with include/emx.h: rerun engine-mlx_b200/rust/gen_sys.py")
            sys.exit(1)
        print(f"sys.rs matches include/emx.h ({len(names)} functions)")
        return
    with open(OUT, "w") as f:
        f.write(text)
    print(f"wrote {OUT} ({len(names)} functions)")


if __name__ == "__main__":
    main()

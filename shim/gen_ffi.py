"""Writes shim/src/ffi.rs from include/*.h: one Rust `extern "C"` declaration per exported function and one `#[repr(C)]`
struct per C struct, so that the binding cannot drift from the headers (tests/test_abi.py re-runs this and compares)."""
import os
import re
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADERS = ["zkb200.h", "zkb200_air.h", "zkb200_prover.h"]
OPAQUE = {"zkb_ctx": "ZkbCtx", "zkb_air_program": "ZkbAirProgram", "zkb_shard_pcs": "ZkbShardPcs"}
STRUCTS = {"zkb_grid": "ZkbGrid", "zkb_dequant_cfg": "ZkbDequantCfg", "zkb_pcs_config": "ZkbPcsConfig",
           "zkb_stark_component": "ZkbStarkComponent", "zkb_air_op": "ZkbAirOp", "zkb_air_stats": "ZkbAirStats", "zkb_rs_group": "ZkbRsGroup",
           "zkb_rs_slot": "ZkbRsSlot", "zkb_rs_program": "ZkbRsProgram", "zkb_rs_tables": "ZkbRsTables", "zkb_rs_mult": "ZkbRsMult",
           "zkb_rs_mults": "ZkbRsMults", "zkb_step_embed_args": "ZkbStepEmbedArgs", "zkb_kv_cache": "ZkbKvCache", "zkb_step_rows": "ZkbStepRows",
           "zkb_step_norm_rope_args": "ZkbStepNormRopeArgs", "zkb_step_attention_args": "ZkbStepAttentionArgs",
           "zkb_step_residual_norm_args": "ZkbStepResidualNormArgs", "zkb_step_gate_args": "ZkbStepGateArgs", "zkb_step_product_args": "ZkbStepProductArgs",
           "zkb_step_logprobs_args": "ZkbStepLogprobsArgs"}
SCALARS = {"int": "i32", "unsigned": "u32", "unsigned int": "u32", "uint32_t": "u32", "int32_t": "i32", "uint64_t": "u64", "int64_t": "i64",
           "unsigned long long": "u64", "size_t": "usize", "float": "f32", "double": "f64", "int8_t": "i8", "uint8_t": "u8",
           "uint16_t": "u16", "unsigned char": "u8", "char": "std::os::raw::c_char", "void": "std::ffi::c_void"}


def strip_comments(text):
    text = re.sub(r"/\*.*?\*/", " ", text, flags=re.S)
    return re.sub(r"//[^\n]*", " ", text)


def base_type(name):
    name = name.strip()
    if name in SCALARS:
        return SCALARS[name]
    if name in OPAQUE:
        return OPAQUE[name]
    if name in STRUCTS:
        return STRUCTS[name]
    raise ValueError(f"unknown C type {name!r}")


def rust_type(ctype):
    """`const uint32_t* const*` -> `*const *const u32` (C declarators read right to left)."""
    c = ctype.strip()
    m = re.match(r"^(.*?)((?:\s*\*\s*(?:const)?)*)$", c)
    head, stars = m.group(1).strip(), m.group(2)
    head_const = bool(re.search(r"\bconst\b", head))
    head = re.sub(r"\bconst\b", "", head).strip()
    levels = re.findall(r"\*\s*(const)?", stars)  # one entry per '*', 'const' if that pointer itself is const
    t = base_type(head)
    pointee_const = head_const
    for k, lv in enumerate(levels):
        t = ("*const " if pointee_const else "*mut ") + t
        pointee_const = lv == "const"
    return t


RENAMED = {"in": "inp", "type": "ty", "ref": "r", "fn": "f", "loop": "lp", "box": "bx"}  # Rust's own words


def parse_param(p):
    p = p.strip()
    if p == "void":
        return None
    m = re.match(r"^(.*?)(\w+)\s*(\[[^\]]*\])?$", p)
    ctype, name, arr = m.group(1).strip(), m.group(2), m.group(3)
    if arr:  # `T x[4]` is `T* x`; a leading const stays with the element
        ctype = ctype + "*"
    name = RENAMED.get(name, name)
    return name, rust_type(ctype)


def parse_struct(name, body):
    fields = []
    for decl in body.split(";"):
        decl = decl.strip()
        if not decl:
            continue
        m = re.match(r"^(.*?)([\w\s,\[\]]+)$", decl)
        first = re.match(r"^((?:const\s+)?(?:unsigned\s+)?\w+(?:\s+long\s+long)?\s*\**)\s*(.*)$", decl)
        ctype, names = first.group(1), first.group(2)
        for nm in names.split(","):
            nm = nm.strip()
            am = re.match(r"^(\w+)\[(\d+)\]$", nm)
            if am:
                fields.append((am.group(1), f"[{rust_type(ctype)}; {am.group(2)}]"))
            else:
                stars = nm.count("*")
                nm = nm.replace("*", "").strip()
                fields.append((RENAMED.get(nm, nm), rust_type(ctype + "*" * stars)))
    return fields


def generate():
    out = ["// Generated by shim/gen_ffi.py from include/zkb200.h, zkb200_air.h and zkb200_prover.h. Do not edit by hand.",
           "// One declaration per exported function of libzkb200.so; status codes as in zkb200.h (0 = ok, < 0 = error).",
           "#![allow(non_snake_case, clippy::too_many_arguments)]", ""]
    for c, r in OPAQUE.items():
        out += [f"#[repr(C)] pub struct {r} {{ _private: [u8; 0] }}  // {c}: opaque"]
    out.append("")
    funcs, seen, no_default = [], set(), set()
    for h in HEADERS:
        text = strip_comments(open(os.path.join(ROOT, "include", h)).read())
        for m in re.finditer(r"typedef\s+struct\s+(\w+)\s*\{(.*?)\}\s*(\w+)\s*;", text, flags=re.S):
            cname = m.group(3)
            if cname in STRUCTS and cname not in seen:
                seen.add(cname)
                fields = parse_struct(cname, m.group(2))
                # raw pointers have no Default; a struct that holds one (directly or through a field struct) is built field by field
                if any("*" in t for _, t in fields):
                    no_default.add(STRUCTS[cname])
                plain = not any("*" in t or t in no_default for _, t in fields)
                out.append("#[repr(C)] #[derive(Copy, Clone, Debug" + (", Default" if plain else "") + ")]")
                out.append(f"pub struct {STRUCTS[cname]} {{")
                for fname, ftype in fields:
                    out.append(f"    pub {fname}: {ftype},")
                out.append("}")
                out.append("")
        for m in re.finditer(r"(?:^|\n)\s*((?:const\s+)?\w+\s*\*?)\s*(zkb_\w+)\s*\(([^;{]*?)\)\s*;", text, flags=re.S):
            ret, name, params = m.group(1).strip(), m.group(2), m.group(3)
            if name in seen:
                continue
            seen.add(name)
            ps = [parse_param(p) for p in re.split(r",(?![^\[]*\])", " ".join(params.split())) if p.strip()]
            ps = [p for p in ps if p]
            rret = rust_type(ret)
            funcs.append((name, ps, rret))
    out.append('extern "C" {')
    for name, ps, rret in funcs:
        args = ", ".join(f"{n}: {t}" for n, t in ps)
        out.append(f"    pub fn {name}({args}) -> {rret};")
    out.append("}")
    out.append("")
    return "\n".join(out), [f[0] for f in funcs]


if __name__ == "__main__":
    text, names = generate()
    path = os.path.join(ROOT, "shim", "src", "ffi.rs")
    if "--check" in sys.argv:
        sys.exit(0 if open(path).read() == text else 1)
    open(path, "w").write(text)
    print(f"{path}: {len(names)} functions")

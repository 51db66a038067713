#!/usr/bin/env python3
"""Generates the Rust FFI declarations and dispatch wrappers of this crate from
the C ABI header (include/runit_hip.h): src/ffi.rs and src/dispatch.rs.

    python gen_bindings.py           # writes both files
    python gen_bindings.py --check   # exits 1 if a committed file is stale

Every header function gets an `extern "C"` declaration; every kernel entry
point (first argument `rt_ctx* ctx`, then device pointers and scalars) also
gets a safe wrapper with the reference's `dispatch::<name>` signature
(crates/kernels/src/dispatch.rs): `&HipContext`, `&Buffer` per device
pointer, scalars as they are.  Context, buffer, event, graph, GGUF and
decode-step functions are wrapped by hand in src/lib.rs.
"""
from __future__ import annotations

import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(HERE, "..", "..", "include", "runit_hip.h")

SCALARS = {"uint32_t": "u32", "uint64_t": "u64", "int": "c_int", "float": "f32", "size_t": "usize",
           "double": "f64", "int64_t": "i64", "uint16_t": "u16"}
POINTEE = {"void": "c_void", "float": "f32", "uint16_t": "u16", "uint32_t": "u32", "uint64_t": "u64",
           "char": "c_char", "int64_t": "i64", "double": "f64", "uint8_t": "u8"}
OPAQUE = {"rt_ctx": "RtCtx", "rt_event": "RtEvent", "rt_graph": "RtGraph", "rt_gguf": "RtGguf",
          "rt_step": "RtStep", "rt_step_model": "RtStepModel", "rt_step_layer": "RtStepLayer",
          "rt_paged_batch": "RtPagedBatch", "rt_logit_rules": "RtLogitRules"}
MANUAL_PREFIXES = ("rt_ctx_", "rt_flush", "rt_last_error", "rt_global_last_error", "rt_malloc",
                   "rt_free", "rt_upload", "rt_download", "rt_memset", "rt_copy_d2d", "rt_event_",
                   "rt_capture_", "rt_graph_", "rt_gguf_", "rt_decode_step_", "rt_has_kernel",
                   "rt_device_cu_count")


def functions(src: str):
    src = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    src = re.sub(r"//[^\n]*", "", src)
    src = re.sub(r"#[^\n]*", "", src)
    for m in re.finditer(r"\b((?:const\s+)?[a-z_0-9]+\s*\**)\s*(rt_[a-z0-9_]+)\s*\(([^)]*)\)\s*;", src):
        ret, name, args = m.group(1).strip(), m.group(2), m.group(3).strip()
        params = [] if args in ("", "void") else [a.strip() for a in args.split(",")]
        yield ret, name, [parse_param(p) for p in params]


def parse_param(p: str):
    """(const, base, stars, name); const is a bool (the pointee's), or for
    pointers to pointers a tuple: per level from the innermost, whether what
    that level points to is const (`const char* const* x`: (True, True))."""
    m = re.match(r"(const\s+)?([a-z_0-9]+)\s*((?:\*\s*(?:const\b\s*)?)*)([a-z_0-9]+)(\[\d+\])?$",
                 p.strip())
    if not m:
        raise ValueError(f"cannot parse parameter '{p}'")
    const, base, name = bool(m.group(1)), m.group(2), m.group(4)
    levels = re.findall(r"\*\s*(const\b)?", m.group(3))
    stars = len(levels)
    if m.group(5):  # an array parameter is a pointer
        stars += 1
        levels.append("")
    if stars > 1:
        const = tuple([const] + [bool(c) for c in levels[:-1]])
    return const, base, stars, name


def rust_type(const, base: str, stars: int) -> str:
    if stars == 0:
        if base in SCALARS:
            return SCALARS[base]
        raise ValueError(base)
    inner = OPAQUE.get(base) or POINTEE.get(base)
    if inner is None:
        raise ValueError(base)
    consts = const if isinstance(const, tuple) else (const,) + (False,) * (stars - 1)
    t = inner
    for i in range(stars):
        t = ("*const " if consts[i] else "*mut ") + t
    return t


def ident(n: str) -> str:
    return n + "_" if n in ("type", "ref", "in", "fn", "match", "mod", "move", "self") else n


def ffi_rs(funcs) -> str:
    out = ["// Generated by gen_bindings.py from include/runit_hip.h; do not edit.",
           "#![allow(non_camel_case_types, clippy::too_many_arguments)]",
           "use std::os::raw::{c_char, c_int, c_void};", "",
           "#[repr(C)] pub struct RtCtx { _p: [u8; 0] }",
           "#[repr(C)] pub struct RtEvent { _p: [u8; 0] }",
           "#[repr(C)] pub struct RtGraph { _p: [u8; 0] }",
           "#[repr(C)] pub struct RtGguf { _p: [u8; 0] }",
           "#[repr(C)] pub struct RtStep { _p: [u8; 0] }", "",
           "/// rt_step_layer (include/runit_hip.h)",
           "#[repr(C)] #[derive(Clone, Copy)]",
           "pub struct RtStepLayer {",
           "    pub wq: *const c_void, pub wk: *const c_void, pub wv: *const c_void,",
           "    pub wo: *const c_void, pub wg: *const c_void, pub wu: *const c_void,",
           "    pub wd: *const c_void,",
           "    pub bq: *const u16, pub bk: *const u16, pub bv: *const u16,",
           "    pub attn_norm: *const f32, pub ffn_norm: *const f32,",
           "    pub k_cache: *mut f32, pub v_cache: *mut f32,",
           "}",
           "/// rt_step_model (include/runit_hip.h)",
           "#[repr(C)]",
           "pub struct RtStepModel {",
           "    pub layers: u32, pub hidden: u32, pub heads: u32, pub kv_heads: u32,",
           "    pub head_dim: u32, pub ff: u32, pub vocab: u32, pub max_seq: u32,",
           "    pub eps: f32, pub theta: f32,",
           "    pub layer: *const RtStepLayer,",
           "    pub token_embd: *const c_void, pub lm_head: *const c_void,",
           "    pub output_norm: *const f32, pub token: *mut u32, pub logits: *mut f32,",
           "}",
           "/// rt_paged_batch (include/runit_hip.h)",
           "#[repr(C)] #[derive(Clone, Copy)]",
           "pub struct RtPagedBatch {",
           "    pub k_pages: *mut c_void, pub v_pages: *mut c_void,",
           "    pub f16: u32, pub num_pages: u32, pub page_size: u32, pub num_kv_heads: u32,",
           "    pub head_dim: u32, pub table_stride: u32, pub n_seqs: u32, pub rows: u32,",
           "    pub page_stride: u64,",
           "    pub table: *const u32, pub row_start: *const u32, pub kv_len: *const u32,",
           "}",
           "/// rt_logit_rules (include/runit_hip.h)",
           "#[repr(C)] #[derive(Clone, Copy)]",
           "pub struct RtLogitRules {",
           "    pub tokens: *const u32, pub token_start: *const u32, pub token_len: *const u32,",
           "    pub prompt_len: *const u32, pub n_tokens: u64,",
           "    pub repetition: *const f32, pub frequency: *const f32, pub presence: *const f32,",
           "    pub bias_ids: *const u32, pub bias_start: *const u32, pub bias_len: *const u32,",
           "    pub bias: *const f32, pub n_bias: u64,",
           "    pub mask: *const u32, pub mask_row: *const u32, pub mask_stride: u64, pub mask_rows: u32,",
           "}", "", "extern \"C\" {"]
    for ret, name, params in funcs:
        args = ", ".join(f"{ident(n)}: {rust_type(c, b, s)}" for c, b, s, n in params)
        if ret == "void":
            r = ""
        elif ret == "int":
            r = " -> c_int"
        else:
            m = re.match(r"(const\s+)?([a-z_0-9]+)\s*(\**)", ret)
            r = " -> " + rust_type(bool(m.group(1)), m.group(2), len(m.group(3)))
        out.append(f"    pub fn {name}({args}){r};")
    out.append("}")
    return "\n".join(out) + "\n"


def dispatch_rs(funcs) -> str:
    out = ["// Generated by gen_bindings.py from include/runit_hip.h; do not edit.",
           "//! The reference's `dispatch::*` surface (crates/kernels/src/dispatch.rs) over the",
           "//! C ABI: one wrapper per kernel entry point, same names and argument order.",
           "#![allow(clippy::too_many_arguments)]",
           "use crate::{ffi, status, Buffer, HipContext, Result};",
           "use std::os::raw::c_void;", ""]
    n = 0
    for ret, name, params in funcs:
        if ret != "int" or name.startswith(MANUAL_PREFIXES):
            continue
        if not params or params[0][1] != "rt_ctx":
            continue
        sig, call = ["ctx: &HipContext"], ["ctx.raw()"]
        ok = True
        for c, b, s, pn in params[1:]:
            if s == 1 and b in POINTEE:
                sig.append(f"{ident(pn)}: &Buffer")
                cast = rust_type(c, b, 1)
                call.append(f"{ident(pn)}.as_ptr() as {cast}")
            elif s == 1 and pn == "batches":  # (with its length)
                sig.append(f"{pn}: &[ffi::{OPAQUE[b]}]")
                call.append(f"{pn}.as_ptr(), {pn}.len() as u32")
            elif pn == "n_batches":
                continue
            elif s == 1 and b in ("rt_paged_batch", "rt_logit_rules"):
                sig.append(f"{ident(pn)}: &ffi::{OPAQUE[b]}")
                call.append(ident(pn))
            elif s == 0 and b in SCALARS:
                sig.append(f"{ident(pn)}: {SCALARS[b]}")
                call.append(ident(pn))
            else:
                ok = False
        if not ok:
            continue
        rname = name[3:]
        out.append(f"pub fn {rname}({', '.join(sig)}) -> Result<()> {{")
        out.append(f"    status(ctx.raw(), unsafe {{ ffi::{name}({', '.join(call)}) }})")
        out.append("}")
        n += 1
    return "\n".join(out) + "\n"


def main() -> int:
    funcs = list(functions(open(HEADER).read()))
    files = {os.path.join(HERE, "src", "ffi.rs"): ffi_rs(funcs),
             os.path.join(HERE, "src", "dispatch.rs"): dispatch_rs(funcs)}
    if "--check" in sys.argv:
        stale = [p for p, txt in files.items() if not os.path.exists(p) or open(p).read() != txt]
        for p in stale:
            print(f"stale: {p}")
        return 1 if stale else 0
    for p, txt in files.items():
        with open(p, "w") as f:
            f.write(txt)
    print(f"{len(funcs)} functions")
    return 0


if __name__ == "__main__":
    sys.exit(main())

#!/usr/bin/env python
"""Generate kernels/cuda_ffi.ts -- the Deno.dlopen symbol table of
libflock_cuda.so -- from include/flock_cuda.h.

    python kernels/gen_ffi.py            # rewrite kernels/cuda_ffi.ts
    python kernels/gen_ffi.py --check    # exit 1 if the committed file is stale

Type map (Deno FFI native types):
  int / int32_t -> "i32", int64_t -> "i64", uint32_t -> "u32",
  float -> "f32", double -> "f64", void (result) -> "void";
  an opaque handle (flock_dev*, flock_model*, ...) -> "pointer";
  any other pointer or array (host data, out-parameters, handle out-slots,
  strings, the flock_layer_config struct) -> "buffer" (a TypedArray);
  a `const char*` result -> "pointer" (read with Deno.UnsafePointerView).
"""
from __future__ import annotations

import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(HERE, "..", "include", "flock_cuda.h")
OUT = os.path.join(HERE, "cuda_ffi.ts")

HANDLES = {"flock_dev", "flock_tensor", "flock_layer", "flock_model", "flock_shard",
           "flock_head", "flock_comm", "flock_gguf", "flock_kv"}
SCALARS = {"int": "i32", "int32_t": "i32", "int64_t": "i64", "uint32_t": "u32",
           "float": "f32", "double": "f64"}
# C scalar sizes/alignments for the struct layout
SIZES = {"int32_t": 4, "float": 4, "double": 8, "int64_t": 8, "uint32_t": 4}


def strip_comments(s: str) -> str:
    s = re.sub(r"/\*.*?\*/", " ", s, flags=re.S)
    return re.sub(r"//[^\n]*", " ", s)


def param_type(decl: str) -> str:
    """Deno FFI type of one C parameter declaration."""
    decl = decl.strip()
    if decl == "void":
        return ""
    array = "[" in decl
    decl = re.sub(r"\[[^\]]*\]", "", decl)
    stars = decl.count("*")
    words = [w for w in re.split(r"[\s*]+", decl) if w and w != "const"]
    base = words[0]
    if array or stars > 1:
        return "buffer"
    if stars == 1:
        return "pointer" if base in HANDLES else "buffer"
    if base not in SCALARS:
        raise ValueError(f"unmapped C type in `{decl}`")
    return SCALARS[base]


def result_type(ret: str) -> str:
    ret = ret.replace("const", "").strip()
    if ret == "int":
        return "i32"
    if ret == "void":
        return "void"
    if ret.replace(" ", "") == "char*":
        return "pointer"
    raise ValueError(f"unmapped result type `{ret}`")


def parse(header: str = HEADER):
    """[(name, [param types], result type, [param names])] in header order,
    the #define constants, and the flock_layer_config fields."""
    src = strip_comments(open(header).read())
    protos = []
    for m in re.finditer(r"FLOCK_API\s+([^;(]*?)\b(flock_\w+)\s*\(([^)]*)\)\s*;", src):
        ret, name, params = m.group(1), m.group(2), m.group(3)
        ps = [p for p in (x.strip() for x in params.split(",")) if p and p != "void"]
        types = [param_type(p) for p in ps]
        names = [re.sub(r"\[[^\]]*\]", "", p).replace("*", " ").split()[-1] for p in ps]
        protos.append((name, types, result_type(ret), names))
    defines = {}
    for m in re.finditer(r"#define\s+(FLOCK_[A-Z0-9_]+)\s+\(?(-?\d+)\)?", src):
        defines[m.group(1)] = int(m.group(2))
    body = re.search(r"typedef struct flock_layer_config\s*\{(.*?)\}\s*flock_layer_config;", src,
                     re.S).group(1)
    fields, off = [], 0
    for line in body.split(";"):
        line = line.strip()
        if not line:
            continue
        ty, nm = line.split()
        size = SIZES[ty]
        off = (off + size - 1) // size * size
        fields.append((nm, ty, off))
        off += size
    align = max(SIZES[t] for _, t, _ in fields)
    struct_size = (off + align - 1) // align * align
    return protos, defines, fields, struct_size


_TS_TYPES = {"int32_t": "Int32", "float": "Float32", "double": "Float64"}


def render(header: str = HEADER) -> str:
    protos, defines, fields, struct_size = parse(header)
    out = []
    w = out.append
    w("// GENERATED by kernels/gen_ffi.py from include/flock_cuda.h -- do not edit.")
    w("// The Deno.dlopen symbol table of libflock_cuda.so, the status and enum")
    w("// constants, and the byte layout of flock_layer_config.  The TypeScript")
    w("// modules beside it (lib.ts, layer.ts, model.ts, shard.ts) keep the")
    w("// reference kernels/ module surface on top of these symbols.")
    w("")
    for k, v in defines.items():
        if k in ("FLOCK_CUDA_H", "FLOCK_API"):
            continue
        w(f"export const {k} = {v};")
    w("")
    w("export const symbols = {")
    for name, types, res, names in protos:
        params = ", ".join(f'"{t}"' for t in types)
        w(f"  // ({', '.join(names)})")
        w(f"  {name}: {{ parameters: [{params}], result: \"{res}\" }},")
    w("} as const;")
    w("")
    w("export type FlockSymbols = typeof symbols;")
    w("export type FlockLib = Deno.DynamicLibrary<FlockSymbols>[\"symbols\"];")
    w("")
    w(f"/** sizeof(flock_layer_config) and each field's byte offset (C layout). */")
    w(f"export const LAYER_CONFIG_BYTES = {struct_size};")
    w("export const LAYER_CONFIG_FIELDS = {")
    for nm, ty, off in fields:
        w(f"  {nm}: {{ offset: {off}, type: \"{ty}\" }},")
    w("} as const;")
    w("")
    w("export type LayerConfigC = { [K in keyof typeof LAYER_CONFIG_FIELDS]: number };")
    w("")
    w("/** Pack a flock_layer_config into the bytes the C ABI reads. */")
    w("export function packLayerConfig(c: LayerConfigC): Uint8Array {")
    w("  const buf = new Uint8Array(LAYER_CONFIG_BYTES);")
    w("  const dv = new DataView(buf.buffer);")
    for nm, ty, off in fields:
        w(f"  dv.set{_TS_TYPES[ty]}({off}, c.{nm}, true);")
    w("  return buf;")
    w("}")
    w("")
    w("let opened: Deno.DynamicLibrary<FlockSymbols> | null = null;")
    w("")
    w("/** dlopen libflock_cuda.so once (FLOCK_LIB overrides the path).  There is")
    w(" *  no fallback: a missing library is an error, not a CPU path. */")
    w("export function flock(path?: string): FlockLib {")
    w("  if (!opened) {")
    w("    const p = path ?? Deno.env.get(\"FLOCK_LIB\") ??")
    w("      new URL(\"../flock_b200/libflock_cuda.so\", import.meta.url).pathname;")
    w("    opened = Deno.dlopen(p, symbols);")
    w("  }")
    w("  return opened.symbols;")
    w("}")
    w("")
    w("/** flock_last_error() as a string. */")
    w("export function lastError(): string {")
    w("  const p = flock().flock_last_error();")
    w("  return p ? new Deno.UnsafePointerView(p).getCString() : \"\";")
    w("}")
    w("")
    w("/** The reference throws `Error`s with named messages; a non-zero status")
    w(" *  becomes the same kind of throw, carrying flock_last_error() and the code. */")
    w("export class FlockError extends Error {")
    w("  constructor(readonly code: number, message: string) {")
    w("    super(message || `flock error ${code}`);")
    w("  }")
    w("}")
    w("")
    w("export function check(rc: number): void {")
    w("  if (rc !== FLOCK_OK) throw new FlockError(rc, lastError());")
    w("}")
    w("")
    w("/** One out-slot for a handle (flock_X** parameters). */")
    w("export function handleSlot(): BigUint64Array {")
    w("  return new BigUint64Array(1);")
    w("}")
    w("")
    w("export function slotPointer(slot: BigUint64Array): Deno.PointerValue {")
    w("  return Deno.UnsafePointer.create(slot[0]);")
    w("}")
    w("")
    w("/** A NUL-terminated UTF-8 string for a `const char*` parameter. */")
    w("export function cstr(s: string): Uint8Array {")
    w("  return new TextEncoder().encode(s + \"\\0\");")
    w("}")
    w("")
    w("/** An array of handles for a `T* const*` parameter. */")
    w("export function pointerArray(ps: Deno.PointerValue[]): BigUint64Array {")
    w("  return BigUint64Array.from(ps.map((p) => BigInt(Deno.UnsafePointer.value(p))));")
    w("}")
    return "\n".join(out) + "\n"


def main() -> int:
    text = render()
    if "--check" in sys.argv:
        cur = open(OUT).read() if os.path.exists(OUT) else ""
        if cur != text:
            print(f"{OUT} is stale: run python kernels/gen_ffi.py", file=sys.stderr)
            return 1
        return 0
    with open(OUT, "w") as f:
        f.write(text)
    print(OUT)
    return 0


if __name__ == "__main__":
    sys.exit(main())

#!/usr/bin/env python
"""Generates integration/PradCuda.cs from include/prad_cuda.h: one [DllImport] per exported function,
the enums and the plain structs, plus the small managed helpers the operation classes use
(status -> exception mapping, a device-matrix handle).  Run it after changing the header:

    python integration/make_bindings.py

tests/test_abi.py checks that the generated file is up to date and names every exported symbol.
The C# file is what a maintainer of the reference adds to the managed project; it cannot be compiled
where this library is built (no .NET toolchain), so its consistency with the header is checked
textually.
"""
from __future__ import annotations

import os
import re

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(HERE, "..", "include", "prad_cuda.h")
OUT = os.path.join(HERE, "PradCuda.cs")

ENUM_NAMES = {"prad_dtype": "DType", "prad_act": "Act", "prad_adam_form": "AdamForm", "prad_op": "Op",
              "prad_tensor_op": "TensorOp"}
STRUCTS = {"prad_device_info_t": "DeviceInfo", "prad_timing_t": "Timing"}
# structs of plain numbers and pointers that a call reads, emitted from the header
IN_STRUCTS = {"prad_scan_t": "Scan", "prad_scan_gradients_t": "ScanGradients"}
# C type -> C# type of a parameter
SCALARS = {"int": "int", "int32_t": "int", "int64_t": "long", "double": "double", "size_t": "UIntPtr", "float": "float",
           "prad_status": "int", "uint64_t": "ulong"}
OUT_SCALARS = {"int*": "out int", "int64_t*": "out long", "double*": "out double", "size_t*": "out UIntPtr"}


def strip_comments(text: str) -> str:
    return re.sub(r"/\*.*?\*/", "", text, flags=re.S)


def pascal(name: str, prefix: str) -> str:
    name = name[len(prefix):] if name.startswith(prefix) else name
    return "".join(p.capitalize() for p in name.lower().split("_"))


def parse_enums(text: str):
    enums = []
    for m in re.finditer(r"typedef\s+enum\s*\{(.*?)\}\s*(\w+)\s*;", text, flags=re.S):
        body, cname = m.group(1), m.group(2)
        items = [(k.strip(), v.strip()) for k, v in re.findall(r"(\w+)\s*=\s*([^,}]+)", body)]
        enums.append((cname, items))
    anon = []
    for m in re.finditer(r"(?<!typedef\s)\benum\s*\{(.*?)\}\s*;", text, flags=re.S):
        anon.append([(k.strip(), v.strip()) for k, v in re.findall(r"(\w+)\s*=\s*([^,}]+)", m.group(1))])
    return enums, anon


def parse_functions(text: str):
    fns = []
    for m in re.finditer(r"\b(prad_status|const char\s*\*)\s+(prad_\w+)\s*\(([^;{]*?)\)\s*;", text, flags=re.S):
        ret, name, args = m.group(1), m.group(2), " ".join(m.group(3).split())
        params = [] if args in ("void", "") else [a.strip() for a in args.split(",")]
        fns.append((ret.replace(" ", ""), name, params))
    return fns


def cs_struct(text: str, cname: str):
    """The fields of a plain struct as C# lines."""
    body = next(b for b, n in re.findall(r"typedef\s+struct\s*\{([^}]*)\}\s*(\w+)\s*;", text) if n == cname)
    lines = []
    for decl in filter(None, (" ".join(d.split()) for d in body.split(";"))):
        m = re.match(r"(?:const )?(\w+)\s*(.*)", decl)
        names = [n.strip() for n in m.group(2).split(",")]
        kind = "IntPtr" if names[0].startswith("*") else SCALARS[m.group(1)]
        fields = []
        for n in names:
            n = n.lstrip("* ")
            parts = [q[0].upper() + q[1:] for q in n.split("_")]
            name = "".join(parts)
            fields.append(name)
        lines.append(f"public {kind} {', '.join(fields)};")
    return lines


def cs_param(p: str) -> str:
    p = p.strip()
    m = re.match(r"(.*?)(\w+)$", p)
    ctype, pname = m.group(1).strip(), m.group(2)
    ctype_n = ctype.replace(" ", "")
    if pname in ("ref", "out", "in", "params", "base", "object", "string", "lock", "event"):
        pname = "@" + pname
    if ctype_n in ("constchar*",):
        return f"[MarshalAs(UnmanagedType.LPStr)] string {pname}"
    for en, cs in ENUM_NAMES.items():
        if ctype_n == en:
            return f"{cs} {pname}"
    for st, cs in STRUCTS.items():
        if ctype_n == st + "*":
            if st == "prad_timing_t":
                return f"[In, Out] {cs}[] {pname}"
            return f"out {cs} {pname}"
    for st, cs in IN_STRUCTS.items():
        if ctype_n == f"const{st}*":
            return f"ref {cs} {pname}"
    if ctype_n in SCALARS:
        return f"{SCALARS[ctype_n]} {pname}"
    if ctype_n in OUT_SCALARS and pname.startswith("out"):
        return f"{OUT_SCALARS[ctype_n]} {pname}"
    if ctype_n in ("prad_ctx**", "prad_graph**", "prad_sequence**", "prad_packed**", "void**") and pname.startswith("out") \
            and not pname.endswith("_host"):
        return f"out IntPtr {pname}"
    if pname.endswith("_host") and "*" in ctype_n:
        # host arrays: of device pointers, of sizes, or a packed host block
        if ctype_n in ("constint64_t*",):
            return f"long[] {pname}"
        if ctype_n in ("constsize_t*",):
            return f"UIntPtr[] {pname}"
        if ctype_n in ("void*const*", "constvoid*const*", "void**"):
            return f"[Out] IntPtr[] {pname}" if pname.startswith("out_") else f"IntPtr[] {pname}"
        return f"IntPtr {pname}"
    if ctype_n in ("constint*",):
        return f"int[] {pname}"
    if ctype_n in ("int*", "double*", "int64_t*"):
        return f"{OUT_SCALARS[ctype_n]} {pname}" if pname.startswith("out") else f"IntPtr {pname}"
    if ctype_n in ("constvoid*const*", "void*const*"):
        return f"IntPtr[] {pname}"
    return f"IntPtr {pname}"        # every other pointer: device memory, handles, 16-byte ids, streams


def generate() -> str:
    text = strip_comments(open(HEADER).read())
    enums, anon = parse_enums(text)
    fns = parse_functions(text)
    out = []
    w = out.append
    w("// <auto-generated> by integration/make_bindings.py from include/prad_cuda.h -- do not edit by hand.")
    w("// P/Invoke surface of libprad_cuda for ParallelReverseAutoDiff (RMAD double / PRADLite float).")
    w("namespace ParallelReverseAutoDiff.RMAD.Cuda")
    w("{")
    w("    using System;")
    w("    using System.Runtime.InteropServices;")
    w("")
    w("    /// <summary>One [DllImport] per function of include/prad_cuda.h.</summary>")
    w("    public static class PradCuda")
    w("    {")
    w('        private const string Lib = "prad_cuda";   // libprad_cuda.so / prad_cuda.dll')
    w("")
    status = next(a for a in anon if any(k == "PRAD_OK" for k, _ in a))
    w("        public enum Status")
    w("        {")
    for k, v in status:
        w(f"            {pascal(k, 'PRAD_')} = {v},")
    w("        }")
    w("")
    for items in anon:
        if items is status:
            continue
        for k, v in items:
            w(f"        public const int {pascal(k, 'PRAD_')} = {v};")
        w("")
    for cname, items in enums:
        cs = ENUM_NAMES[cname]
        prefix = os.path.commonprefix([k for k, _ in items])
        prefix = prefix[: prefix.rfind("_") + 1]
        w(f"        public enum {cs}")
        w("        {")
        for k, v in items:
            w(f"            {pascal(k, prefix)} = {v},")
        w("        }")
        w("")
    for m in re.finditer(r"#define\s+(PRAD_\w+)\s+(\d+)", text):
        w(f"        public const int {pascal(m.group(1), 'PRAD_')} = {m.group(2)};")
    w("")
    w("        [StructLayout(LayoutKind.Sequential, CharSet = CharSet.Ansi)]")
    w("        public struct DeviceInfo")
    w("        {")
    w("            public int Device, SmCount, CcMajor, CcMinor, L2Bytes, SmemPerBlockOptin, SmClockKhz, MemClockKhz;")
    w("            public ulong TotalBytes, FreeBytes, ScratchBytes;")
    w("            [MarshalAs(UnmanagedType.ByValTStr, SizeConst = 64)] public string Name;")
    w("        }")
    w("")
    w("        [StructLayout(LayoutKind.Sequential, CharSet = CharSet.Ansi)]")
    w("        public struct Timing")
    w("        {")
    w("            [MarshalAs(UnmanagedType.ByValTStr, SizeConst = 48)] public string Label;")
    w("            public double Milliseconds;")
    w("            public long Launches;")
    w("        }")
    w("")
    for cname, cs in IN_STRUCTS.items():
        w("        [StructLayout(LayoutKind.Sequential)]")
        w(f"        public struct {cs}")
        w("        {")
        for line in cs_struct(text, cname):
            w(f"            {line}")
        w("        }")
        w("")
    for ret, name, params in fns:
        cs_ret = "IntPtr" if ret.startswith("constchar") else "int"
        w(f"        [DllImport(Lib, CallingConvention = CallingConvention.Cdecl)]")
        w(f"        public static extern {cs_ret} {name}({', '.join(cs_param(p) for p in params)});")
        w("")
    w("        /// <summary>Maps a status to the exception the managed operation would have thrown.</summary>")
    w("        public static void Check(int status)")
    w("        {")
    w("            if (status == 0)")
    w("            {")
    w("                return;")
    w("            }")
    w("")
    w('            string msg = Marshal.PtrToStringAnsi(prad_last_error()) ?? "libprad_cuda error";')
    w("            switch ((Status)status)")
    w("            {")
    w("                case Status.ErrShape: throw new InvalidOperationException(msg);           // MatrixMultiplyOperation.cs:59-62")
    w("                case Status.ErrNotInitialized: throw new CudaNotInitializedException();    // GpuMatrixMultiplyOperation.cs:115-118")
    w("                case Status.ErrInvalid: throw new ArgumentException(msg);")
    w("                case Status.ErrOom: throw new OutOfMemoryException(msg);")
    w("                case Status.ErrTimeout: throw new TimeoutException(msg);                   // visitor TimeoutInMinutes")
    w('                default: throw new InvalidOperationException("CUDA failure: " + msg);     // CudaBlas.cs:251-256')
    w("            }")
    w("        }")
    w("    }")
    w("")
    w("    /// <summary>A dense row-major matrix (or DeepMatrix: depth consecutive matrices) resident on the device.</summary>")
    w("    public sealed class DeviceMatrix : IDisposable")
    w("    {")
    w("        public DeviceMatrix(IntPtr ctx, PradCuda.DType dtype, int rows, int cols, int depth = 1)")
    w("        {")
    w("            this.Ctx = ctx;")
    w("            this.DType = dtype;")
    w("            this.Rows = rows;")
    w("            this.Cols = cols;")
    w("            this.Depth = depth;")
    w("            PradCuda.Check(PradCuda.prad_alloc(ctx, (UIntPtr)this.Bytes, out IntPtr p));")
    w("            this.Ptr = p;")
    w("        }")
    w("")
    w("        public IntPtr Ctx { get; }")
    w("")
    w("        public IntPtr Ptr { get; private set; }")
    w("")
    w("        public PradCuda.DType DType { get; }")
    w("")
    w("        public int Rows { get; }")
    w("")
    w("        public int Cols { get; }")
    w("")
    w("        public int Depth { get; }")
    w("")
    w("        public int ElementSize => this.DType == PradCuda.DType.F64 ? 8 : 4;")
    w("")
    w("        public ulong Bytes => (ulong)this.Rows * (ulong)this.Cols * (ulong)this.Depth * (ulong)this.ElementSize;")
    w("")
    w("        /// <summary>Uploads a jagged double[][] / float[][] (pinned row by row) with one call.</summary>")
    w("        public void Upload(Array[] rows)")
    w("        {")
    w("            var handles = new GCHandle[rows.Length];")
    w("            var ptrs = new IntPtr[rows.Length];")
    w("            try")
    w("            {")
    w("                for (int i = 0; i < rows.Length; ++i)")
    w("                {")
    w("                    handles[i] = GCHandle.Alloc(rows[i], GCHandleType.Pinned);")
    w("                    ptrs[i] = handles[i].AddrOfPinnedObject();")
    w("                }")
    w("")
    w("                PradCuda.Check(PradCuda.prad_upload_rows(this.Ctx, this.Ptr, ptrs, rows.Length, (UIntPtr)((ulong)this.Cols * (ulong)this.ElementSize)));")
    w("                PradCuda.Check(PradCuda.prad_sync(this.Ctx));")
    w("            }")
    w("            finally")
    w("            {")
    w("                foreach (var h in handles)")
    w("                {")
    w("                    if (h.IsAllocated)")
    w("                    {")
    w("                        h.Free();")
    w("                    }")
    w("                }")
    w("            }")
    w("        }")
    w("")
    w("        /// <summary>Downloads into a jagged array of the same shape (blocks until the copy is done).</summary>")
    w("        public void Download(Array[] rows)")
    w("        {")
    w("            var handles = new GCHandle[rows.Length];")
    w("            var ptrs = new IntPtr[rows.Length];")
    w("            try")
    w("            {")
    w("                for (int i = 0; i < rows.Length; ++i)")
    w("                {")
    w("                    handles[i] = GCHandle.Alloc(rows[i], GCHandleType.Pinned);")
    w("                    ptrs[i] = handles[i].AddrOfPinnedObject();")
    w("                }")
    w("")
    w("                PradCuda.Check(PradCuda.prad_download_rows(this.Ctx, ptrs, this.Ptr, rows.Length, (UIntPtr)((ulong)this.Cols * (ulong)this.ElementSize)));")
    w("            }")
    w("            finally")
    w("            {")
    w("                foreach (var h in handles)")
    w("                {")
    w("                    if (h.IsAllocated)")
    w("                    {")
    w("                        h.Free();")
    w("                    }")
    w("                }")
    w("            }")
    w("        }")
    w("")
    w("        public void Dispose()")
    w("        {")
    w("            if (this.Ptr != IntPtr.Zero)")
    w("            {")
    w("                PradCuda.prad_free(this.Ctx, this.Ptr);")
    w("                this.Ptr = IntPtr.Zero;")
    w("            }")
    w("        }")
    w("    }")
    w("}")
    return "\n".join(out) + "\n"


def declared_functions():
    return [name for _, name, _ in parse_functions(strip_comments(open(HEADER).read()))]


if __name__ == "__main__":
    text = generate()
    with open(OUT, "w") as f:
        f.write(text)
    print(f"{OUT}: {len(declared_functions())} functions")

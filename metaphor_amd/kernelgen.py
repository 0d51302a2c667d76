"""Kernel generation and device compilation for the gfx950 library.

Plays the part of the reference's build-time generator and compiler driver
(file_gen.zig:200-340, script_compiler.zig:151-314, build.zig:11-45), re-targeted to HIP:

* the fused elementwise chains listed in ``chains.json`` are turned into forward and reverse
  kernel sources first (``chaingen.py``: expression -> HIP source by reverse-mode differentiation);
* every source in ``csrc/hipcc_src`` is written against the placeholder type ``Scalar`` and
  is replicated for r16, r32 and r64 by textual substitution into ``csrc/hipcc_trg``
  (file_gen.zig:217-244);
* the ``extern "C" void launch_*`` prototypes of all targets are scraped into
  ``include/kernel_decls.h`` (file_gen.zig:264-288), together with the comment block that
  precedes each launcher in its source;
* targets are compiled with ``hipcc --offload-arch=gfx950`` (the reference shells out to
  ``nvcc --gpu-architecture=sm_89``, script_compiler.zig:151-187) and archived into
  ``lib/mp_kernels.a`` (script_compiler.zig:189-201); the same objects are also linked into
  ``lib/libmp_kernels.so`` for FFI callers that cannot link a static archive;
* ``csrc/device_utils.hip`` becomes ``lib/libdev_utils.so`` (script_compiler.zig:281-314).

Nothing here needs a GPU: hipcc cross-compiles.
"""
import concurrent.futures
import json
import os
import re
import shutil
import subprocess
import sys

PKG = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
SRC_DIR = os.path.join(CSRC, "hipcc_src")
TRG_DIR = os.path.join(CSRC, "hipcc_trg")
OBJ_DIR = os.path.join(CSRC, "obj")
LIB_DIR = os.path.join(PKG, "lib")
INCLUDE = os.path.join(ROOT, "include")
DECLS = os.path.join(INCLUDE, "kernel_decls.h")
CONFIG = os.path.join(PKG, "config.json")

SCALARS = ("r16", "r32", "r64")
DECL_RE = re.compile(r'extern "C" void \w+\s?\([^)]+\)')
LAUNCH_RE = re.compile(r"void (launch_\w+)")


def load_config():
    """``config.json``: compiler path and architecture (reference: config.json:1-4 and
    script_compiler.zig:19-72, which insists on an ``sm_`` prefix; here it must be ``gfx``)."""
    with open(CONFIG) as f:
        cfg = json.load(f)
    arch = cfg["gpu-architecture"]
    if not arch.startswith("gfx"):
        raise ValueError(f"gpu-architecture must start with 'gfx', got {arch!r}")
    hipcc = cfg.get("hipcc-path", "/opt/rocm/bin/hipcc")
    if not os.path.exists(hipcc):
        found = shutil.which("hipcc")
        if not found:
            raise FileNotFoundError("hipcc not found")
        hipcc = found
    return hipcc, arch


# the matrix products and the per-stream handle come from rocBLAS (the reference links cuBLAS, build.zig:139)
BLAS_LINK = ["-L/opt/rocm/lib", "-lrocblas"]


def device_flags(arch):
    return [
        f"--offload-arch={arch}", "-O3", "-std=c++20", "-fPIC",
        # packed fp32 arithmetic stays off for every device object of this library
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        "-Wno-unused-command-line-argument",
        f"-I{INCLUDE}", f"-I{CSRC}",
    ]


def collect_sources():
    return sorted(f for f in os.listdir(SRC_DIR) if f.endswith(".hip"))


def _newer(src, dst):
    return not os.path.exists(dst) or os.path.getmtime(src) > os.path.getmtime(dst)


def _header_mtime():
    times = [os.path.getmtime(os.path.join(CSRC, f)) for f in os.listdir(CSRC) if f.endswith(".h")]
    times += [os.path.getmtime(os.path.join(INCLUDE, f)) for f in ("tensor_types.h", "device_utils.h")]
    return max(times)


def make_device_kernels(force=False):
    """Scalar replication (file_gen.zig:200-262). Returns the stems whose target changed."""
    os.makedirs(TRG_DIR, exist_ok=True)
    changed = []
    for name in collect_sources():
        src, trg = os.path.join(SRC_DIR, name), os.path.join(TRG_DIR, name)
        if not (force or _newer(src, trg)):
            continue
        with open(src) as f:
            text = f.read()
        if "Scalar" not in text:
            raise ValueError(f"{name}: a kernel source must be written against `Scalar`")
        copies = [text.replace("Scalar", s) for s in SCALARS]
        with open(trg, "w") as f:
            f.write("\n".join(copies))
        changed.append(name[:-4])
    return changed


def _leading_comment(text, pos):
    """The block of // lines that ends right above character offset pos."""
    lines = text[:pos].splitlines()
    block = []
    for line in reversed(lines):
        if line.startswith("//"):
            block.append(line)
        else:
            break
    return list(reversed(block))


def make_kernel_declarations():
    """Scrape every launcher prototype into include/kernel_decls.h (file_gen.zig:264-288)."""
    out = [
        "/* GENERATED by metaphor_amd/kernelgen.py from metaphor_amd/csrc/hipcc_src -- do not edit.",
        " *",
        " * Kernel launchers of the drop-in boundary. Every stem S exports launch_S_r16, launch_S_r32",
        " * and launch_S_r64 with one C signature: device pointers as void*, scalars as double, sizes",
        " * as len_t, the StreamContext by value as the last argument, no return value and no error",
        " * channel (a failure prints and exits). This is the shape of the reference's generated",
        " * src/cuda/kernel_decls.h:11-436; the comment above each group names what it replaces.",
        " * Launchers only enqueue work on the context's stream and allocate nothing.",
        " */",
        "#ifndef __KERNEL_DECLS_H__",
        "#define __KERNEL_DECLS_H__",
        "",
        '#include "tensor_types.h"',
        "",
        "#if defined(__cplusplus)",
        '    #define EXTERN_C extern "C"',
        "#else",
        "    #define EXTERN_C extern",
        "#endif",
        "",
    ]
    for name in collect_sources():
        with open(os.path.join(SRC_DIR, name)) as f:
            text = f.read()
        for m in DECL_RE.finditer(text):
            out.extend(c.replace("//", "/*", 1) + " */" for c in _leading_comment(text, m.start()))
            proto = m.group(0).replace('extern "C"', "EXTERN_C")
            for s in SCALARS:
                out.append(proto.replace("Scalar", s) + ";")
            out.append("")
    out += [
        "/* Not per-dtype; defined in metaphor_amd/csrc/kernel_support.hip. */",
        "/* Bytes of caller-owned scratch for launch_rmsnorm_ij_j_reverse_<dtype> on an [m, n] problem;",
        " * dtype is the dispatch key 0 = r16, 1 = r32, 2 = r64 (src/core/scalar.zig:35-40). The reference",
        " * sizes per-stream scratch on the host the same way (src/core/utils.zig:20-36). */",
        "EXTERN_C len_t mpRmsnormReverseScratchBytes(len_t dtype, len_t m, len_t n);",
        "/* Bytes of caller-owned scratch launch_softmax_ij_j_<dtype> can use on an [m, n] problem (0 when a row",
        " * fits one workgroup; NULL scratch is allowed and costs a second read of long rows). Rows shared by",
        " * several workgroups exchange their partial results through words that, where it can, the library keeps",
        " * in device memory of its own, one region per workspace address and problem geometry: the workspace is",
        " * then the key that keeps launches apart (launches that may overlap in time must be given different",
        " * workspaces, as they must when the words are in the workspace itself) and is not written. */",
        "EXTERN_C len_t mpSoftmaxScratchBytes(len_t dtype, len_t m, len_t n);",
        "EXTERN_C len_t mpSoftmaxReverseScratchBytes(len_t dtype, len_t m, len_t n);",
        "EXTERN_C len_t mpReduceScratchBytes(len_t dtype, len_t m, len_t n);",
        "EXTERN_C len_t mpRmsnormScratchBytes(len_t dtype, len_t m, len_t n);",
        "EXTERN_C len_t mpLayernormReverseScratchBytes(len_t dtype, len_t m, len_t n);",
        "EXTERN_C len_t mpEmbeddingReverseScratchBytes(len_t dtype, len_t v, len_t m, len_t n);",
        "EXTERN_C len_t mpGradientNormScratchBytes(len_t dtype, len_t count);",
        "/* launch_rmsnorm_ij_j_reverse_r32 without the scratch argument, for callers that cannot allocate a",
        " * workspace (code under HIP graph capture, serving loops, harnesses that forbid hipMalloc): the partial",
        " * gain rows go into a 16 MiB device array that the library holds on every GPU it runs on. It has no",
        " * counterpart in the reference. Same kernels, bit-identical results. Returns 0 after enqueueing, 1",
        " * (message on stderr, nothing enqueued) when [m, n] needs more than the 16 MiB: min(m, 2 * CUs) * n * 4",
        " * bytes, so rows of up to 4194304 / min(m, 2 * CUs) elements fit, 8192 on the MI355X's 256 compute",
        " * units. Calls no hipMalloc / hipFree; its first call on a device looks the array's address up (make",
        " * that call before a graph capture starts). All calls on one GPU share the array: calls that overlap in",
        " * time on one GPU race, and a call on another stream than the one before prints one warning saying so. */",
        "EXTERN_C int mpRmsnormReverseR32NoAlloc(const void* src, const void* gain, const void* dst_grads, void* src_grads, void* gain_grads, double eps, double alpha, len_t m, len_t n, StreamContext stream);",
        "",
        "#endif",
        "",
    ]
    text = "\n".join(out)
    old = open(DECLS).read() if os.path.exists(DECLS) else None
    if old != text:
        with open(DECLS, "w") as f:
            f.write(text)


def kernel_table():
    """{stem: [launch_stem_r16, launch_stem_r32, launch_stem_r64]} — the content of the
    reference's generated src/core/kernels.zig dispatch arrays (file_gen.zig:298-328)."""
    table = {}
    for name in collect_sources():
        with open(os.path.join(SRC_DIR, name)) as f:
            text = f.read()
        launchers = LAUNCH_RE.findall(text)
        if len(launchers) != 1:
            raise ValueError(f"{name}: exactly one launcher per source file, found {launchers}")
        table[name[:-4]] = [launchers[0].replace("Scalar", s) for s in SCALARS]
    return table


HOST_DIR = os.path.join(PKG, "host")


def make_kernel_overloads():
    """Dispatch arrays for the C++ host side: host/kernels.hpp, the counterpart of the
    reference's generated src/core/kernels.zig (file_gen.zig:28-35, 298-328)."""
    out = [
        "// GENERATED by metaphor_amd/kernelgen.py -- do not edit.",
        "// One three-entry dispatch array per kernel stem, indexed by the dtype key",
        "// (0 = r16, 1 = r32, 2 = r64), as src/core/kernels.zig holds them; calling the array is",
        "// src/core/root.zig:36-43 (invoke).",
        "#ifndef MP_HOST_KERNELS_HPP",
        "#define MP_HOST_KERNELS_HPP",
        "",
        "#include <cstddef>",
        "",
        '#include "kernel_decls.h"',
        "",
        "namespace mp {",
        "[[noreturn]] void panic(const char* what);",
        "namespace kernels {",
        "",
        "template <class Fn> struct DispatchArray {",
        "  Fn* fn[3];",
        "  template <class... Args> void operator()(size_t key, Args... args) const {",
        '    if (key > 2) panic("invoke: dtype key out of range");',
        "    fn[key](args...);",
        "  }",
        "};",
        "",
    ]
    for stem, arr in kernel_table().items():
        out.append(f"inline const DispatchArray<decltype({arr[0]})> {stem}{{{{{', '.join(arr)}}}}};")
    out += ["", "}  // namespace kernels", "}  // namespace mp", "", "#endif", ""]
    text = "\n".join(out)
    path = os.path.join(HOST_DIR, "kernels.hpp")
    if not os.path.exists(path) or open(path).read() != text:
        with open(path, "w") as f:
            f.write(text)


def build_host(force=False):
    """The C++ host library (graph, ops, fusion) and its check program, with g++."""
    make_kernel_overloads()
    lib = os.path.join(LIB_DIR, "libmetaphor_host.so")
    exe = os.path.join(LIB_DIR, "host_check")
    srcs = [os.path.join(HOST_DIR, f) for f in ("metaphor.cpp", "metaphor.hpp", "kernels.hpp", "chains.hpp", "host_check.cpp")]
    srcs += [os.path.join(LIB_DIR, "libmp_kernels.so"), os.path.join(LIB_DIR, "libmp_fusion.so"), DECLS,
             os.path.join(INCLUDE, "chain_fusion.h")]
    stale = force or any(_newer(s, lib) for s in srcs) or any(_newer(s, exe) for s in srcs)
    if stale:
        common = ["-std=c++17", "-O2", "-fPIC", "-Wall", "-Wextra", f"-I{INCLUDE}", f"-I{HOST_DIR}"]
        link = [f"-L{LIB_DIR}", "-lmp_kernels", "-lmp_fusion", "-ldev_utils", "-Wl,-rpath,$ORIGIN"]
        _run(["g++", "-shared", "-o", lib, os.path.join(HOST_DIR, "metaphor.cpp")] + common + link)
        _run(["g++", "-o", exe, os.path.join(HOST_DIR, "host_check.cpp")] + common +
             [f"-L{LIB_DIR}", "-lmetaphor_host"] + link[1:])
    return {"host": lib, "host_check": exe}


def _run(cmd):
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(" ".join(cmd) + "\n" + res.stdout + res.stderr)
        raise RuntimeError(f"command failed: {cmd[0]} ... {cmd[-1]}")
    return res


def _compile(hipcc, arch, src, obj, extra=()):
    _run([hipcc, "-c", src, "-o", obj] + device_flags(arch) + list(extra))
    return obj


# Sources compiled once (no Scalar replication) into the shipped library.
SUPPORT_SOURCES = ("kernel_support.hip", "noalloc_entry.hip")

# The test build: the row launchers and the workspace-size functions compiled with
# -DMP_DIAGNOSTICS, which turns the row regime and the cluster tuning from constants into
# process-wide switches behind mpSetRowRegime / mpSetClusterTuning / mpSetClusterDeep. They go into a library of
# their own that only the parity tests load; the shipped library exports neither function.
DIAG_STEMS = ("softmax_ij_j", "softmax_ij_j_reverse", "rmsnorm_ij_j", "rmsnorm_ij_j_reverse")
DIAG_FLAGS = ("-DMP_DIAGNOSTICS",)


# Headers a chain compiled at run time includes; chain_fusion.hip carries their text.
CHAIN_HEADERS = ((INCLUDE, "tensor_types.h"), (CSRC, "kernel_header.h"), (CSRC, "elementwise.h"))


def make_chain_headers():
    """obj/chain_headers.inc: the text of the headers above as string literals, so that the
    run-time compiler sees exactly what the library's own kernels were built from."""
    names, texts = [], []
    for folder, name in CHAIN_HEADERS:
        with open(os.path.join(folder, name)) as f:
            text = f.read()
        if ')MPHDR"' in text:
            raise ValueError(f"{name} contains the raw-string delimiter")
        names.append(f'"{name}"')
        texts.append('R"MPHDR(' + text + ')MPHDR"')
    out = ("// GENERATED by metaphor_amd/kernelgen.py -- do not edit.\n"
           f"static const int CHAIN_HEADER_COUNT = {len(names)};\n"
           "static const char* const CHAIN_HEADER_NAMES[] = {" + ", ".join(names) + "};\n"
           "static const char* const CHAIN_HEADER_TEXT[] = {\n" + ",\n".join(texts) + "};\n")
    path = os.path.join(OBJ_DIR, "chain_headers.inc")
    if not os.path.exists(path) or open(path).read() != out:
        with open(path, "w") as f:
            f.write(out)
    return path


def build_fusion(hipcc, arch, force=False):
    """lib/libmp_fusion.so: elementwise expressions compiled at run time (chain_fusion.hip)."""
    inc = make_chain_headers()
    src = os.path.join(CSRC, "chain_fusion.hip")
    lib = os.path.join(LIB_DIR, "libmp_fusion.so")
    deps = [src, inc, os.path.join(INCLUDE, "chain_fusion.h")]
    if force or any(_newer(d, lib) for d in deps):
        _run([hipcc, "--shared", "-o", lib, src] + device_flags(arch) +
             [f"-I{OBJ_DIR}", f'-DMP_GPU_ARCH="{arch}"', "-L/opt/rocm/lib", "-lhiprtc"])
    return lib


def build(force=False, jobs=None, verbose=False):
    """Generate, compile and link everything. force=True recompiles every object."""
    hipcc, arch = load_config()
    os.makedirs(OBJ_DIR, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    from . import chaingen
    chaingen.generate()  # fused elementwise chains of chains.json -> hipcc_src/*.hip, host/chains.hpp
    make_device_kernels(force)
    make_kernel_declarations()
    kernel_table()  # validates one launcher per file

    hdr = _header_mtime()
    todo = []
    objs = []
    for name in collect_sources():
        trg = os.path.join(TRG_DIR, name)
        obj = os.path.join(OBJ_DIR, name[:-4] + ".o")
        objs.append(obj)
        if force or _newer(trg, obj) or hdr > os.path.getmtime(obj):
            todo.append((trg, obj))
    for name in SUPPORT_SOURCES:
        src, obj = os.path.join(CSRC, name), os.path.join(OBJ_DIR, name[:-4] + ".o")
        objs.append(obj)
        if force or _newer(src, obj) or hdr > os.path.getmtime(obj):
            todo.append((src, obj))
    diag_objs = []
    for src in [os.path.join(TRG_DIR, stem + ".hip") for stem in DIAG_STEMS] + [os.path.join(CSRC, "kernel_support.hip")]:
        obj = os.path.join(OBJ_DIR, "diag_" + os.path.basename(src)[:-4] + ".o")
        diag_objs.append(obj)
        if force or _newer(src, obj) or hdr > os.path.getmtime(obj):
            todo.append((src, obj, DIAG_FLAGS))

    jobs = jobs or min(8, os.cpu_count() or 1)
    if todo:
        if verbose:
            print(f"[kernelgen] hipcc --offload-arch={arch}: {len(todo)} objects, {jobs} jobs", flush=True)
        with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as pool:
            for obj in pool.map(lambda p: _compile(hipcc, arch, *p), todo):
                if verbose:
                    print(f"[kernelgen]   {os.path.basename(obj)}", flush=True)

    archive = os.path.join(LIB_DIR, "mp_kernels.a")
    shared = os.path.join(LIB_DIR, "libmp_kernels.so")
    diag = os.path.join(LIB_DIR, "libmp_kernels_diag.so")
    if todo or not all(os.path.exists(p) for p in (archive, shared, diag)):
        if os.path.exists(archive):
            os.remove(archive)
        _run(["ar", "-rcs", archive] + objs)
        _run([hipcc, "--shared", "-o", shared] + objs + [f"--offload-arch={arch}", "-fPIC"] + BLAS_LINK)
        # -Bsymbolic: the test build defines the same symbols as the shipped library; its own calls
        # must reach its own definitions when both are loaded into one process
        _run([hipcc, "--shared", "-o", diag] + diag_objs + [f"--offload-arch={arch}", "-fPIC", "-Wl,-Bsymbolic"])

    utils_src = os.path.join(CSRC, "device_utils.hip")
    utils_so = os.path.join(LIB_DIR, "libdev_utils.so")
    if force or _newer(utils_src, utils_so) or hdr > os.path.getmtime(utils_so):
        _run([hipcc, "--shared", "-o", utils_so, utils_src] + device_flags(arch) + BLAS_LINK)
    # measurement only: plain passes with a workload's stream mix, loaded by bench.py alone
    probe_src = os.path.join(CSRC, "stream_probe.hip")
    probe_so = os.path.join(LIB_DIR, "libmp_probe.so")
    if force or _newer(probe_src, probe_so) or hdr > os.path.getmtime(probe_so):
        _run([hipcc, "--shared", "-o", probe_so, probe_src] + device_flags(arch))
    libs = {"archive": archive, "kernels": shared, "kernels_diag": diag, "device_utils": utils_so,
            "probe": probe_so, "fusion": build_fusion(hipcc, arch, force)}
    libs.update(build_host(force))  # links the fusion library: after it
    return libs


if __name__ == "__main__":
    libs = build(force="--force" in sys.argv, verbose=True)
    for k, v in libs.items():
        print(f"{k}: {v}")

"""Builds libcust_opapi.so (the aclnn C-ABI over the gfx950 HIP kernels) in-tree with hipcc.

    python ops-transformer_amd/build.py [--force | --sanitize]

hipcc cross-compiles for gfx950 without a GPU.  Objects go to ops-transformer_amd/build/, the library to
ops-transformer_amd/lib/libcust_opapi.so — the file name the reference's dlsym-based binder searches first
(common/include/fallback/fallback.h:79-135 in the reference).
"""
import concurrent.futures
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OBJ_DIR = os.path.join(HERE, "build")
LIB_DIR = os.path.join(HERE, "lib")
LIB_PATH = os.path.join(LIB_DIR, "libcust_opapi.so")
BINDING_PATH = os.path.join(LIB_DIR, "opapi_torch.so")  # the Python module that reads torch's tensors; the library itself knows nothing of torch
EXPORTS = os.path.join(CSRC, "exports.map")  # linker version script: only the C entry points leave the library

SOURCES = [
    "acl_runtime.cpp",
    "moe_gating_top_k_softmax_v2.hip",
    "moe_add_rms_norm_quant.hip",
    "moe_router_logits.hip",
    "moe_gating_top_k_grouped.hip",
    "moe_init_routing.hip",
    "grouped_gemm_i8.hip",
    "grouped_gemm_i8_int32.hip",
    "grouped_gemm_i8_dequant.hip",
    "grouped_gemm_i8_swiglu.hip",
    "grouped_gemm_i8_int32_tail.hip",
    "grouped_gemm_i8_dequant_tail.hip",
    "grouped_gemm_i8_swiglu_tail.hip",
    "grouped_gemm_i8_slim_plain.hip",
    "grouped_gemm_i8_slim_swiglu.hip",
    "grouped_matmul_swiglu_quant.hip",
    "grouped_matmul_v4.hip",
    "grouped_matmul_finalize_routing.hip",
    "moe_finalize_routing_v2.hip",
    "moe_ffn_forward.hip",
    "packed_operators.hip",
    "calibration_copy.hip",
]

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

COMMON_FLAGS = [
    "-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden", "--offload-arch=gfx950",
    "-ffp-contract=off",
    # packed-fp32 instructions stay off for all device code
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wall", "-Wno-unused-command-line-argument", "-Wno-unknown-attributes",
    "-I", os.path.join(ROOT, "include"), "-I", CSRC,
]


# The translation units that hold the LDS-DMA kernels (grouped_gemm_i8_kernels.h instantiated per epilogue): their device
# assembly goes through the guards below whenever they are compiled.
RING_SOURCES = ("grouped_gemm_i8_int32.hip", "grouped_gemm_i8_dequant.hip", "grouped_gemm_i8_swiglu.hip",
                "grouped_gemm_i8_int32_tail.hip", "grouped_gemm_i8_dequant_tail.hip", "grouped_gemm_i8_swiglu_tail.hip",
                "grouped_gemm_i8_slim_plain.hip", "grouped_gemm_i8_slim_swiglu.hip")

# The LDS-DMA loads of grouped_gemm_i8_kernels.h set m0 in an inline-assembly statement and count outstanding loads by hand,
# which leans on how this compiler schedules around such statements.  The kernels were validated (bit-exact suites on
# the GPU) with the compiler named here; another one has to be validated again before its build is trusted:
# OPAPI_ALLOW_UNVALIDATED_COMPILER=1 lets the build through so that the suites can be run.
VALIDATED_COMPILERS = ("roc-7.2.0",)
LDS_DMA_LOADS = ("global_load_lds_dwordx4", "global_load_lds_dword")  # operand chunks, scales


def compiler_version():
    out = subprocess.run([HIPCC, "--version"], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True).stdout
    for line in out.splitlines():
        if "clang version" in line:
            return line.strip()
    return out.strip().splitlines()[0] if out.strip() else "unknown"


def check_compiler():
    version = compiler_version()
    if any(tag in version for tag in VALIDATED_COMPILERS) or os.environ.get("OPAPI_ALLOW_UNVALIDATED_COMPILER") == "1":
        return version
    raise RuntimeError(
        "hipcc reports '%s', but the LDS-DMA kernels of grouped_gemm_i8_kernels.h (m0 set in inline assembly, hand-counted "
        "s_waitcnt vmcnt) were validated with %s only. Set OPAPI_ALLOW_UNVALIDATED_COMPILER=1 to build anyway, run "
        "`pytest tests -m gpu` on an MI355X, and add the compiler to VALIDATED_COMPILERS in %s when the suites are green."
        % (version, " / ".join(VALIDATED_COMPILERS), os.path.abspath(__file__)))


def check_lds_dma_assembly(asm_path):
    """Build-time guard on the device assembly of the GEMM kernel units: every instruction that writes m0 must be the
    `s_mov_b32 m0, sN` of an LDS-DMA statement, i.e. be followed at once by its global_load_lds_dword[x4], and every such
    load must be preceded by its own m0 write.  A compiler that puts anything between the two, or writes m0 for a
    purpose of its own inside these kernels, fails the build instead of producing kernels that read stale tiles."""
    lines = [l.split(";")[0].strip() for l in open(asm_path)]
    lines = [l for l in lines if l and not l.startswith(".") and not l.endswith(":")]
    loads = pairs = 0
    for i, l in enumerate(lines):
        fields = l.replace(",", " ").split()
        writes_m0 = len(fields) > 1 and fields[1] == "m0" and not fields[0].startswith(("s_cmp", "s_bitcmp"))
        if writes_m0:
            nxt = lines[i + 1] if i + 1 < len(lines) else ""
            if fields[0] != "s_mov_b32" or nxt.split(" ")[0] not in LDS_DMA_LOADS:
                raise RuntimeError("%s: m0 is written outside an LDS-DMA pair: '%s' followed by '%s'" % (asm_path, l, nxt))
            pairs += 1
        if l.startswith("global_load_lds_"):
            loads += 1
            prev = lines[i - 1] if i > 0 else ""
            if not prev.startswith("s_mov_b32 m0,"):
                raise RuntimeError("%s: an LDS-DMA load does not follow its m0 write: '%s' after '%s'" % (asm_path, l, prev))
    if loads == 0 or loads != pairs:
        raise RuntimeError("%s: %d LDS-DMA loads, %d m0 writes" % (asm_path, loads, pairs))
    return loads


def check_ring_kernel_codegen(asm_path):
    """Second build-time guard on the device assembly of the GEMM kernel units, for three properties of the generated code
    that the kernels' speed and exactness rest on and that a compiler can change without any test noticing at once:
      * no LDS-ring kernel (StreamGemmKernel, MixedGemmKernel, SlimGemmKernel) uses scratch memory -- a spilled register is reloaded inside the tile loop;
      * no generic (flat) memory instruction: one still in flight makes the compiler drain vmcnt, DMAs included, in
        front of every LDS read;
      * no mixed-precision multiply-add (v_fma_mix*, v_mad_mix*): that is a product and its fp16 conversion merged into
        one rounding, where the reference rounds the product to fp32 first.
    Returns the number of ring kernels checked."""
    text = open(asm_path).read()
    for bad in ("v_fma_mix", "v_mad_mix"):
        if bad in text:
            raise RuntimeError("%s: the compiler merged a multiply with an fp16 conversion (%s*)" % (asm_path, bad))
    for bad in ("flat_load_", "flat_store_", "flat_atomic_"):
        if bad in text:
            raise RuntimeError("%s: generic memory instruction (%s*) in the GEMM kernels" % (asm_path, bad))
    checked = 0
    for block in text.split(".amdhsa_kernel ")[1:]:
        name = block.split()[0]
        if not any(ring in name for ring in ("StreamGemmKernel", "MixedGemmKernel", "SlimGemmKernel")):
            continue
        fields = dict(l.split()[:2] for l in block.split(".end_amdhsa_kernel")[0].splitlines()[1:] if len(l.split()) >= 2)
        if int(fields.get(".amdhsa_private_segment_fixed_size", "0")) != 0:
            raise RuntimeError("%s: %s spills %s bytes per lane to scratch" %
                               (asm_path, name, fields[".amdhsa_private_segment_fixed_size"]))
        checked += 1
    if checked == 0:
        raise RuntimeError("%s: no LDS-ring kernel found" % asm_path)
    return checked


def check_ring_barrier_waits(asm_path):
    """Third build-time guard: a barrier among a ring kernel's matrix instructions frees LDS buffers for DMAs that the compiler does
    not see, so the wave's reads of them have to have been waited for.  In the device assembly of StreamGemmKernel and
    MixedGemmKernel, going back from every s_barrier inside a basic block that multiplies, a wait for LDS (lgkmcnt of at most four:
    the reads of the rows' second half, which the barrier does not free) has to come before any LDS read.  Nor may such a block wait for
    every memory request (vmcnt(0)): the compiler does so where it believes a register's load still pending, and the DMAs in flight are
    then drained in every k-step.
    Returns the number of barriers checked."""
    checked = 0
    for body in open(asm_path).read().split("; -- Begin function ")[1:]:
        name = body.split()[0]
        if not any(ring in name for ring in ("StreamGemmKernel", "MixedGemmKernel")):
            continue
        block = []
        for l in body.split("; -- End function")[0].splitlines() + ["end:"]:
            l = l.split(";")[0].strip()
            if l.endswith(":") or l.startswith("s_cbranch"):  # a basic block ends
                multiplies = any(i.startswith("v_mfma") for i in block)
                if multiplies and any(i.startswith("s_waitcnt") and "vmcnt(0)" in i for i in block):
                    raise RuntimeError("%s: %s drains its DMAs in the k loop" % (asm_path, name))
                for at in [i for i, ins in enumerate(block) if multiplies and ins.startswith("s_barrier")]:
                    settled = False
                    for ins in reversed(block[:at]):
                        if ins.startswith("s_waitcnt") and "lgkmcnt(" in ins and int(ins.split("lgkmcnt(")[1].split(")")[0]) <= 4:
                            settled = True
                            break
                        if ins.startswith("ds_read"):
                            break
                    if not settled:
                        raise RuntimeError("%s: %s: a barrier frees LDS buffers whose reads have not been waited for" % (asm_path, name))
                    checked += 1
                block = []
            elif l and not l.startswith("."):
                block.append(l)
    return checked


def _headers():
    out = []
    for base in (CSRC, os.path.join(ROOT, "include")):
        for d, _, files in os.walk(base):
            out += [os.path.join(d, f) for f in files if f.endswith(".h")]
    return out


def _compile(src, force):
    obj = os.path.join(OBJ_DIR, os.path.splitext(src)[0] + ".o")
    src_path = os.path.join(CSRC, src)
    deps = [src_path] + _headers()
    # Whenever this one is recompiled its device assembly is kept for the m0 / LDS-DMA and code-generation guards below
    # (-save-temps adds little to a compile that takes minutes).  OPAPI_ASM_GUARD=0 skips them for a timing experiment;
    # the object is then marked unguarded and a later build without the variable compiles it again.
    guard_stamp = obj + ".guard-passed"
    unguarded_ok = os.environ.get("OPAPI_ASM_GUARD") == "0"
    is_ring_source = src in RING_SOURCES
    if is_ring_source and not force and not unguarded_ok and os.path.exists(obj) and not os.path.exists(guard_stamp):
        os.remove(obj)  # built without the guards: not to be linked
    if not force and os.path.exists(obj) and all(os.path.getmtime(obj) >= os.path.getmtime(d) for d in deps):
        return obj, False
    guarded = is_ring_source and not unguarded_ok
    if is_ring_source and os.path.exists(guard_stamp):
        os.remove(guard_stamp)
    if is_ring_source and not guarded:
        sys.stderr.write("build.py: OPAPI_ASM_GUARD=0 -- %s is compiled WITHOUT the assembly guards\n" % src)
    cmd = [HIPCC] + COMMON_FLAGS + (["-save-temps=obj"] if guarded else []) + \
          (["-x", "hip"] if src.endswith(".cpp") else []) + ["-c", src_path, "-o", obj]
    res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    noise = "is not a recognized feature for this target"
    log = "\n".join(l for l in res.stdout.splitlines() if noise not in l)
    if res.returncode != 0:
        raise RuntimeError("hipcc failed for %s:\n%s" % (src, log))
    if guarded:
        stem = os.path.join(OBJ_DIR, os.path.splitext(src)[0])
        try:
            check_lds_dma_assembly(stem + "-hip-amdgcn-amd-amdhsa-gfx950.s")
            check_ring_kernel_codegen(stem + "-hip-amdgcn-amd-amdhsa-gfx950.s")
            if "slim" not in src and check_ring_barrier_waits(stem + "-hip-amdgcn-amd-amdhsa-gfx950.s") == 0:
                raise RuntimeError("%s: no barrier found among the matrix instructions" % src)
        except Exception:
            os.remove(obj)  # never leave an object behind that the guard refused
            raise
        finally:
            for f in os.listdir(OBJ_DIR):  # the other intermediate files of -save-temps
                if f.startswith((os.path.splitext(src)[0] + "-", src + "-")):
                    os.remove(os.path.join(OBJ_DIR, f))
        open(guard_stamp, "w").write("m0 / LDS-DMA pairing and ring-kernel code generation checked\n")
    if log.strip():
        sys.stderr.write(log + "\n")
    return obj, True


# Host-side sanitizer build (AddressSanitizer + UndefinedBehaviorSanitizer on the host pass only; device code is compiled
# as usual and GPU sanitizers are never involved).  The per-epilogue GEMM units, whose host part is a few lines of dispatch
# around minutes of kernel compilation, are linked from the regular build.
SANITIZED_LIB_PATH = os.path.join(LIB_DIR, "sanitized", "libcust_opapi.so")
SANITIZE_FLAGS = ["-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
                  "-Xarch_host", "-fno-sanitize-recover=undefined", "-Xarch_host", "-fno-omit-frame-pointer", "-g"]
UNSANITIZED = set(RING_SOURCES)


def sanitizer_runtime():
    """Path of the shared AddressSanitizer runtime of the compiler behind hipcc (to preload into an uninstrumented host
    program such as python)."""
    clang = os.path.join(os.path.dirname(os.path.realpath(HIPCC)), "..", "lib", "llvm", "bin", "clang")
    if not os.path.exists(clang):
        clang = "/opt/rocm/lib/llvm/bin/clang"
    return subprocess.check_output([clang, "-print-file-name=libclang_rt.asan-x86_64.so"], text=True).strip()


def build_sanitized(jobs=None):
    """Builds lib/sanitized/libcust_opapi.so: same sources, host code instrumented.  Returns its path."""
    build()  # the regular objects (those of the GEMM kernel units are reused)
    obj_dir = os.path.join(OBJ_DIR, "sanitized")
    os.makedirs(obj_dir, exist_ok=True)
    os.makedirs(os.path.dirname(SANITIZED_LIB_PATH), exist_ok=True)

    def one(src):
        if src in UNSANITIZED:
            return os.path.join(OBJ_DIR, os.path.splitext(src)[0] + ".o")
        obj = os.path.join(obj_dir, os.path.splitext(src)[0] + ".o")
        src_path = os.path.join(CSRC, src)
        deps = [src_path] + _headers()
        if os.path.exists(obj) and all(os.path.getmtime(obj) >= os.path.getmtime(d) for d in deps):
            return obj
        flags = [f for f in COMMON_FLAGS if f != "-O3"] + ["-O1"] + SANITIZE_FLAGS
        cmd = [HIPCC] + flags + (["-x", "hip"] if src.endswith(".cpp") else []) + ["-c", src_path, "-o", obj]
        res = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        if res.returncode != 0:
            raise RuntimeError("hipcc (sanitized) failed for %s:\n%s" % (src, res.stdout))
        return obj

    jobs = jobs or min(len(SOURCES), os.cpu_count() or 1)
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as pool:
        objs = list(pool.map(one, SOURCES))
    cmd = [HIPCC, "-shared", "-fPIC", "--offload-arch=gfx950", "-fsanitize=address", "-fsanitize=undefined",
           "-shared-libsan", "-Wl,--version-script=" + EXPORTS, "-o", SANITIZED_LIB_PATH] + objs
    subprocess.check_call(cmd)
    return SANITIZED_LIB_PATH


def build_binding(force=False):
    """Compiles the Python module (host code only) against the installed torch's headers.  Returns its path, None where there is no torch, no g++ or
    no Python headers: callers of the C interface need none of them, and the operators that the module serves say that it is missing."""
    import shutil
    import sysconfig

    try:
        import torch
    except ImportError:
        sys.stderr.write("torch is not installed: opapi_torch.so is not built\n")
        return None
    for there, what in [(shutil.which("g++"), "g++"), (os.path.exists(os.path.join(sysconfig.get_paths()["include"], "Python.h")), "Python.h")]:
        if not there:
            sys.stderr.write("%s is not installed: opapi_torch.so is not built\n" % what)
            return None
    src = os.path.join(CSRC, "torch_binding.cpp")
    deps = [src, os.path.abspath(__file__), torch.version.__file__] + _headers()
    if not force and os.path.exists(BINDING_PATH) and all(os.path.getmtime(BINDING_PATH) >= os.path.getmtime(d) for d in deps):
        return BINDING_PATH
    base = os.path.dirname(torch.__file__)
    include = [os.path.join(base, "include"), os.path.join(base, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"],
               os.path.join(ROOT, "include")]
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-D_GLIBCXX_USE_CXX11_ABI=%d" % int(torch.compiled_with_cxx11_abi())]
    cmd += ["-isystem" + d for d in include[:3]] + ["-I" + include[3], src, "-o", BINDING_PATH, "-L" + os.path.join(base, "lib")]
    subprocess.check_call(cmd + ["-ltorch_python", "-ltorch_cpu", "-lc10"])
    return BINDING_PATH


def build(force=False, jobs=None):
    """Compile every source for gfx950 and link the shared library, and the Python module over it.  Returns the library's path."""
    check_compiler()
    os.makedirs(OBJ_DIR, exist_ok=True)
    os.makedirs(LIB_DIR, exist_ok=True)
    jobs = jobs or min(len(SOURCES), os.cpu_count() or 1)
    with concurrent.futures.ThreadPoolExecutor(max_workers=jobs) as pool:
        binding = pool.submit(build_binding, force)
        results = list(pool.map(lambda s: _compile(s, force), SOURCES))
    objs = [o for o, _ in results]
    if any(r for _, r in results) or not os.path.exists(LIB_PATH) or any(os.path.getmtime(LIB_PATH) < os.path.getmtime(f) for f in objs + [EXPORTS]):
        cmd = [HIPCC, "-shared", "-fPIC", "--offload-arch=gfx950", "-Wl,--version-script=" + EXPORTS, "-o", LIB_PATH] + objs
        subprocess.check_call(cmd)
    binding.result()  # the library does not wait for it
    return LIB_PATH


if __name__ == "__main__":
    print(build_sanitized() if "--sanitize" in sys.argv else build(force="--force" in sys.argv))

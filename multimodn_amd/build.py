"""Build libmmn_hip.so in-tree with hipcc for gfx950.  `python -m multimodn_amd.build`."""
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
SRC = os.path.join(CSRC, "mmn_kernels.hip")
INC = os.path.join(os.path.dirname(HERE), "include")
OUT = os.path.join(HERE, "libmmn_hip.so")
BINDING = os.path.join(HERE, "_binding.so")
OBJ = os.path.join(os.path.dirname(HERE), "build")
HEADERS = ("mmn_hip.h", "mmn_sequence.h")
#: the library's translation units, compiled side by side
UNITS = ("mmn_kernels.hip", "mmn_sequence.hip", "mmn_scan.hip")
#: packed 32-bit float operations off: some of their forms have given wrong results on this hardware
_NO_PACKED = ("-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops")


def hipcc_path() -> str:
    for cand in (shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found (need ROCm)")


def source_files():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".hip", ".inc", ".cpp"))) + [os.path.join(INC, h) for h in HEADERS]


def source_hash() -> str:
    """sha256 over the library's sources (names and contents, fixed order), first 16 hex digits: baked into the library at
    build time (`mmn_source_hash()`), compared by `needs_build()` and by `hip.load()` - a library that was not built from
    the sources next to it does not load (modification times say nothing on a box that received the tree by copy)."""
    import hashlib
    h = hashlib.sha256()
    for p in source_files():
        h.update(os.path.basename(p).encode() + b"\0")
        with open(p, "rb") as f:
            h.update(f.read())
        h.update(b"\0")
    return h.hexdigest()[:16]


def built_hash(path: str = OUT):
    """What `mmn_source_hash()` of an existing library says (None: no such library / symbol).  Asked in a CHILD process:
    loading a stale library here and the rebuilt one afterwards would leave two copies mapped in the building process."""
    if not os.path.exists(path):
        return None
    code = ("import ctypes,sys\n"
            "try:\n"
            "    lib = ctypes.CDLL(sys.argv[1]); fn = lib.mmn_source_hash; fn.restype = ctypes.c_char_p; print(fn().decode())\n"
            "except (OSError, AttributeError):\n"
            "    print('')\n")
    try:
        out = subprocess.run([sys.executable, "-c", code, path], capture_output=True, text=True, timeout=120)
    except (OSError, subprocess.TimeoutExpired):
        return None
    h = out.stdout.strip().splitlines()[-1] if out.stdout.strip() else ""
    return h or None


def needs_build() -> bool:
    if not os.path.exists(OUT) or not os.path.exists(BINDING) or built_hash() != source_hash():
        return True
    with open(BINDING, "rb") as f:                         # (the hash is a string constant of the binding)
        return source_hash().encode() not in f.read()


def binding_command():
    """g++ on csrc/binding.cpp against this interpreter's torch."""
    import sysconfig
    import torch
    from torch.utils import cpp_extension
    lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    inc = [f"-I{p}" for p in (*cpp_extension.include_paths(), sysconfig.get_paths()["include"], INC)]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-w", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            "-DTORCH_EXTENSION_NAME=_binding", f'-DMMN_SOURCE_HASH="{source_hash()}"', *inc, os.path.join(CSRC, "binding.cpp"),
            f"-L{lib}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-ldl", f"-Wl,-rpath,{lib}", "-o", BINDING]


def build(force: bool = False, verbose: bool = False, only=None) -> str:
    """Compile and link.  `only`: compile these units and take the others' objects as they are (a developer's shortcut)."""
    if not force and not needs_build():
        return OUT
    # -amdgpu-mfma-vgpr-form: accumulators stay in VGPRs (gfx950's register file is unified).  With AGPR accumulators
    # hipcc rotated k_wgrad's sixteen accumulator tiles through v_accvgpr_read / _write pairs in every unrolled loop
    # body (reads that wait for the MFMA that produced the tile): k_wgrad 18.1 -> 17.5 us, the step -1.4 us.
    flags = ["-O3", "--offload-arch=gfx950", "-std=c++17", "-fPIC", "-mllvm", "-amdgpu-mfma-vgpr-form", *_NO_PACKED, f"-I{INC}"]
    os.makedirs(OBJ, exist_ok=True)
    objects, running = [], []
    for unit in UNITS:
        obj = os.path.join(OBJ, unit.replace(".hip", ".o"))
        cmd = [hipcc_path(), *flags, "-c", os.path.join(CSRC, unit), "-o", obj]
        if unit == "mmn_sequence.hip":                     # (the unit that says what the library was built from: a quick one)
            cmd.insert(1, f'-DMMN_SOURCE_HASH="{source_hash()}"')
        objects.append(obj)
        if only is not None and unit not in only and unit != "mmn_sequence.hip" and os.path.exists(obj):
            continue
        if verbose:
            print(" ".join(cmd), flush=True)
        running.append((unit, subprocess.Popen(cmd)))
    if verbose:
        print(" ".join(binding_command()), flush=True)
    running.append(("binding.cpp", subprocess.Popen(binding_command())))
    failed = [unit for unit, p in running if p.wait() != 0]
    if failed:
        raise RuntimeError(f"the compiler failed on {', '.join(failed)}")
    subprocess.run([hipcc_path(), "--offload-arch=gfx950", "-shared", "-fPIC", *objects, "-o", OUT], check=True)
    return OUT


if __name__ == "__main__":
    units = [a for a in sys.argv[1:] if a in UNITS]
    print(build(force="--force" in sys.argv or bool(units), verbose=True, only=units or None))

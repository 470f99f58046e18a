"""Builds the backend in place: the gfx950 code objects (hipcc --genco), embedded as byte
arrays into libslm_hip.so together with the host runtime (runtime.cpp, the C ABI of
include/slm_hip.h), the model twin (model.cpp, include/slm_model.h) and the fixed device
scratch of the allocation-free entry points (scratch.hip, a HIP translation unit of its own).

    python slm.use_amd/build.py          # or __graft_entry__.build()
"""

import os
import subprocess
import sys
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libslm_hip.so"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

# Device code: gfx950 only; expressions round as written (no contraction into FMA), IEEE
# division and sqrt, and no packed-FP32 instructions. MFMA accumulators in ordinary vector
# registers: the 48-row prompt GEMMs otherwise kept them in accumulator registers and moved
# them to vector registers for every slice sum (vector instructions beside the MFMAs, which
# never overlap them).
DEVICE_FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off",
    "-fhip-fp32-correctly-rounded-divide-sqrt",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-mllvm", "-amdgpu-mfma-vgpr-form=1",
]
HOST_FLAGS = ["-O2", "-std=c++17", "-fPIC", "-ffp-contract=off", "-Wall", "-Wno-unused-result"]


def run(cmd):
    out = subprocess.run(cmd, capture_output=True, text=True)
    if out.returncode != 0:
        raise RuntimeError(f"{' '.join(map(str, cmd))}\n{out.stdout}{out.stderr}")
    return out


def embed(co: Path, dst: Path, name: str):
    data = co.read_bytes()
    rows = []
    for i in range(0, len(data), 24):
        rows.append(",".join(str(b) for b in data[i:i + 24]))
    dst.write_text(
        "// generated by slm.use_amd/build.py from a gfx950 code object\n"
        "#include <stddef.h>\n"
        "extern \"C\" {\n"
        f"extern const unsigned char {name}[{len(data)}];\n"
        f"extern const size_t {name}_size;\n"
        f"alignas(4096) const unsigned char {name}[{len(data)}] = {{\n"
        + ",\n".join(rows) + "\n};\n"
        f"const size_t {name}_size = {len(data)};\n"
        "}\n")


def build(verbose: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    blobs = []
    for src, name in (("kernels", "slm_code_object"), ("batch", "slm_batch_object")):
        co = BUILD / f"{src}.co"
        run([HIPCC, "--genco", *DEVICE_FLAGS, str(CSRC / f"{src}.hip"), "-o", str(co)])
        blobs.append(BUILD / f"{src}_blob.cpp")
        embed(co, blobs[-1], name)
    objs = [BUILD / "scratch.o"]
    run([HIPCC, "-c", "-fPIC", *DEVICE_FLAGS, str(CSRC / "scratch.hip"), "-o", str(objs[0])])
    for src in (CSRC / "runtime.cpp", CSRC / "model.cpp", *blobs):
        objs.append(BUILD / (src.stem + ".o"))
        run([HIPCC, *HOST_FLAGS, "-c", "-I", str(ROOT / "include"), str(src), "-o", str(objs[-1])])
    tmp = LIB.with_suffix(".so.tmp")
    run([HIPCC, "-shared", "-fPIC", *map(str, objs), "-o", str(tmp)])
    os.replace(tmp, LIB)
    if verbose:
        sizes = ", ".join(f"{p.name} {p.stat().st_size}" for p in sorted(BUILD.glob("*.co")))
        print(f"built {LIB} ({LIB.stat().st_size} bytes; {sizes})")
    return LIB


if __name__ == "__main__":
    build(verbose=True)
    sys.exit(0)

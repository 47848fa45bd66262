"""Builds libturbine_mi355.so (the gfx950 kernels + C ABI) in-tree with hipcc.

Usage: ``python -m iree_turbine_amd.build``.  hipcc cross-compiles for gfx950 without a GPU.
"""

from __future__ import annotations

import os
import shutil
import re
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

CSRC = Path(__file__).resolve().parent / "csrc"
LIB_NAME = "libturbine_mi355.so"
LIB_PATH = CSRC / LIB_NAME
HOST_PATH = CSRC / "mi355_host_ops.so"
SOURCES = ["capi.hip", "gemm_f16_nt.hip", "flash_attn_fwd.hip", "paged_decode.hip", "gemm_mxfp4.hip", "gemm_mxfp8.hip", "gemm_mxfp6.hip", "quantize_mxfp4.hip", "quantize_mxfp6.hip", "paged_layout.hip", "rope.hip", "paged_tree.hip", "verify_draft.hip", "calibrate.hip"]

# -packed-fp32-ops: keep the compiler from forming v_pk_{add,mul,fma}_f32.
HIPCC_FLAGS = [
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-command-line-argument",
    "-Wno-unknown-warning-option",
]


def _hipcc() -> str:
    exe = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(exe):
        raise RuntimeError("hipcc not found; cannot build the gfx950 kernel library")
    return exe


# Kernels that load into registers by inline assembly with hand-placed waits ("staged", "skinny"): the compiler does
# not know that such a register may still be receiving its load, so it must never move one -- no spill to scratch,
# no spill of any other kind, and no change of the register budget that a different occupancy would bring.  The
# expected occupancy (waves per SIMD) is pinned per kernel family; a compiler that allocates differently fails the
# build instead of producing a kernel that stores a register before its data has arrived.
# The prefill and decode kernels place waits for LDS transpose reads and loads by hand as well, and are built for two
# waves per SIMD (a spill there also costs the time their schedules were tuned for).
NO_SPILL_KERNELS = ("staged", "skinny", "gemm_f16_nt_stream", "gemm_mxfp4_stream", "gemm_mxfp8_stream", "fa_fwd_d128_pipe",
                    "fa_fwd_d128_m16", "fa_fwd_d128_walk", "paged_decode_phase0", "paged_tree_kernel", "gemm_f16_nt_pipelined", "gemm_mxfp4_tiled")
EXPECTED_OCCUPANCY = {"staged": 1, "gemm_f16_nt_stream": 1, "gemm_mxfp4_stream": 1, "gemm_mxfp8_stream": 1, "gemm_f16_nt_skinnyI": 7,
                      "gemm_mxfp4_skinny": 2, "fa_fwd_d128_pipe": 2, "fa_fwd_d128_m16": 2, "fa_fwd_d128_walk": 2, "paged_decode_phase0": 2,
                      "paged_tree_kernel": 2}
_USAGE_FLAG = "-Rpass-analysis=kernel-resource-usage"


def _remark_int(text: str) -> int:
    """The value of a 'Field [unit]: N [-Rpass...]' remark (a 'file:line:col:' prefix may precede the field)."""
    m = re.search(r"(?:\]|[A-Za-z])\s*:\s*(\d+)\s*(?:\[|$)", text)
    if m is None:
        raise RuntimeError(f"cannot read the value of the resource remark {text!r}")
    return int(m.group(1))


def _check_resource_remarks(stderr: str) -> list[str]:
    """Returns the remark-free stderr lines; raises if a kernel named in NO_SPILL_KERNELS uses scratch, spills a
    vector register, or is built for another occupancy than EXPECTED_OCCUPANCY pins for it."""
    rest, name = [], None
    for line in stderr.splitlines():
        if _USAGE_FLAG not in line and "remark:" not in line:
            # the source excerpt and caret lines that follow a remark
            if name is not None and (line.lstrip().startswith("|") or line.strip()[:1].isdigit() or line.strip() in ("^", "")):
                continue
            rest.append(line)
            continue
        text = line.split("remark:", 1)[1]
        if "Function Name:" in text:
            name = text.split("Function Name:", 1)[1].split("[")[0].strip()
            continue
        if name is None or not any(k in name for k in NO_SPILL_KERNELS):
            continue
        if "ScratchSize" in text and _remark_int(text):
            raise RuntimeError(f"kernel {name} spills ({_remark_int(text)} bytes of scratch per lane); it must fit its registers")
        if "VGPRs Spill" in text and _remark_int(text):
            raise RuntimeError(f"kernel {name} spills {_remark_int(text)} vector registers; it must fit its registers")
        if "Occupancy" in text:
            families = [f for f in EXPECTED_OCCUPANCY if f in name]
            if families:
                want = EXPECTED_OCCUPANCY[max(families, key=len)]  # the longest name that matches: skinny64 before skinny
                if _remark_int(text) != want:
                    raise RuntimeError(f"kernel {name} is built for {_remark_int(text)} waves per SIMD, expected {want}: its "
                                       "register allocation changed; check the hand-placed waits against the new code")
    return rest


def _run(cmd: list[str]) -> None:
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"command failed ({proc.returncode}): {' '.join(cmd)}\n{proc.stdout}\n{proc.stderr}")
    # the host pass warns that it does not know the packed-fp32 feature; that is expected
    noise = ("packed-fp32-ops", "is not a recognized feature")
    for line in _check_resource_remarks(proc.stderr):
        if line.strip() and not any(n in line for n in noise):
            print(line, file=sys.stderr)


def build_library(verbose: bool = True, save_temps: bool = False, defines: tuple[str, ...] = (), out: Path | None = None) -> Path:
    """Compiles every kernel source and links the shared library.  Always recompiles.

    `defines` (e.g. ("MI355_ABLATE_NO_LOADS",), the timing-only switches of csrc/common.hpp) and `out` build a second
    library beside the product one, with its own object directory; the product library is the call without them."""
    hipcc = _hipcc()
    lib_path = Path(out).resolve() if out is not None else LIB_PATH
    if defines and lib_path == LIB_PATH:
        raise ValueError("a build with ablation switches needs its own --out path: it must not replace the product library")
    obj_dir = CSRC / "build" if lib_path == LIB_PATH else lib_path.parent / (lib_path.stem + "_obj")
    obj_dir.mkdir(parents=True, exist_ok=True)
    objs = [obj_dir / (Path(s).stem + ".o") for s in SOURCES]

    def compile_one(pair):
        src, obj = pair
        cmd = [hipcc, *HIPCC_FLAGS, *(f"-D{d}" for d in defines), _USAGE_FLAG, "-c", str(CSRC / src), "-o", str(obj)]
        if save_temps:
            cmd += ["-save-temps=obj"]
        _run(cmd)
        return obj

    with ThreadPoolExecutor(max_workers=min(len(SOURCES), os.cpu_count() or 4)) as pool:
        list(pool.map(compile_one, zip(SOURCES, objs)))
    _run([hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", str(lib_path), *map(str, objs)])
    if verbose:
        print(f"built {lib_path} ({lib_path.stat().st_size} bytes)" + (f" with {' '.join(defines)}" if defines else ""))
    return lib_path


def build_host_ops(verbose: bool = True) -> Path:
    """Compiles the extension module with the host side of the serving operators (host code only, against torch's headers)."""
    import sysconfig

    import torch

    root = Path(torch.__file__).parent
    _run([shutil.which("g++") or "g++", "-std=c++17", "-O2", "-Wall", "-fPIC", "-shared", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
          "-isystem", str(root / "include"), "-isystem", str(root / "include/torch/csrc/api/include"), "-isystem", sysconfig.get_paths()["include"],
          "-isystem", str(Path(_hipcc()).resolve().parent.parent / "include"), str(CSRC / "host_ops.cpp"), "-o", str(HOST_PATH), "-L" + str(root / "lib"),
          "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10", "-lc10_hip"])
    if verbose:
        print(f"built {HOST_PATH} ({HOST_PATH.stat().st_size} bytes)")
    return HOST_PATH


PROBES = ["lds_read_patterns.hip", "load_rate.hip", "mfma_load_bubble.hip", "hbm_read_patterns.hip"]


def build_probes(verbose: bool = True) -> list[Path]:
    """Compiles the stand-alone measurement programs of csrc/probes/ (no Python, no library: each prints a table)."""
    hipcc = _hipcc()
    out_dir = CSRC / "probes" / "bin"
    out_dir.mkdir(exist_ok=True)

    def one(src):
        exe = out_dir / Path(src).stem
        _run([hipcc, *[f for f in HIPCC_FLAGS if f != "-fPIC"], str(CSRC / "probes" / src), "-o", str(exe)])
        return exe

    with ThreadPoolExecutor(max_workers=len(PROBES)) as pool:
        exes = list(pool.map(one, PROBES))
    if verbose:
        print("built " + ", ".join(str(e) for e in exes))
    return exes


if __name__ == "__main__":
    import argparse

    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--save-temps", action="store_true")
    ap.add_argument("-D", dest="defines", action="append", default=[], metavar="MI355_ABLATE_...",
                    help="a timing-only ablation switch (csrc/common.hpp); needs --out")
    ap.add_argument("--out", default=None, help="path of the library to write (default: the product library in csrc/)")
    ap.add_argument("--probes", action="store_true", help="also build the measurement programs of csrc/probes/")
    a = ap.parse_args()
    if a.probes:
        build_probes()
    build_library(save_temps=a.save_temps, defines=tuple(a.defines), out=a.out)
    if a.out is None:
        build_host_ops()

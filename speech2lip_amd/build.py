"""Build libs2l_hip.so (gfx950) in-tree with hipcc.  Cross-compiles without a GPU."""
from __future__ import annotations

import json
import os
import re
import shutil
import subprocess
import sys
import warnings

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
HEADER = os.path.join(PKG, "..", "include", "s2l_hip.h")
LIB = os.path.join(PKG, "libs2l_hip.so")
REF_LIB = os.path.join(PKG, "libs2l_hip_ref.so")      # the same ABI + the non-default kernel forms (-DS2L_WITH_REFERENCE_KERNELS): tests / tools only
TORCH_OPS_SOURCE = "linear_autograd.cpp"
TORCH_OPS = os.path.join(PKG, "_linear_ops.so")        # the autograd node of the dense layer: C++ against torch, calls LIB through its C ABI
RESOURCES = os.path.join(PKG, "kernel_resources.json")      # per-kernel registers / spills / scratch / LDS of the last build
SOURCES = ["pack.hip", "frontend.hip", "rows.hip", "render.hip", "ensemble.hip", "train.hip", "composite.hip", "unet.hip", "warp.hip", "syncnet.hip", "lpips.hip", "syncchain.hip", "train_bf16.hip", "quant.hip", "render16.hip", "convh.hip",
           "linear.hip", "linear_f32.hip", "linear_bf16.hip", "linear_f16.hip", "orthogonalize.hip"]
# translation units that differ in the reference library: the split convolution's generated-assembly form (conv16.hip, its dispatch in
# unet.hip) and the four-wave / alternating-roles forms of the half-width convolution (convh.hip).  Every other object is shared.
REF_SOURCES = ["unet.hip", "convh.hip", "conv16.hip"]
# -ffp-contract=off: parity needs the reference's separate roundings (x*y then +z); FMAs are explicit fmaf()
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fno-gpu-rdc", "-ffp-contract=off", "-Wall",
         "-Wno-unused-function", "-Rpass-analysis=kernel-resource-usage"]
# without packed fp32 instructions (v_pk_add / mul / fma_f32), whose generated forms are not relied on here; the sources that are not listed hold
# such instructions in their own assembly text and are compiled as they were measured
SCALAR_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
SOURCE_FLAGS = {s: SCALAR_FP32 for s in SOURCES if s.startswith(("linear", "orthogonalize"))}
SOURCE_FLAGS["orthogonalize.hip"] = SCALAR_FP32 + ["-mllvm", "-amdgpu-kernarg-preload-count=16"]      # its launches are short: see its place_of
_REMARK = re.compile(r"remark:\s+(Function Name|VGPRs|AGPRs|ScratchSize \[bytes/lane\]|SGPRs Spill|VGPRs Spill|LDS Size \[bytes/block\]|"
                     r"Occupancy \[waves/SIMD\]):\s*(\S+)")


def _parse_resources(text: str) -> dict:
    """{kernel symbol: {vgprs, agprs, scratch, sgpr_spill, vgpr_spill, lds, occupancy}} from -Rpass-analysis=kernel-resource-usage.
    Several kernels wait with COUNTED vmcnt on requests the compiler does not know as memory operations (render, bf16 forward /
    backward bodies, conv3x3_split_kernel): a register spill to scratch would be an uncounted vector-memory operation inside their
    loops, so tests/test_abi_and_host.py checks this table for zero scratch."""
    out, cur = {}, None
    keys = {"VGPRs": "vgprs", "AGPRs": "agprs", "ScratchSize [bytes/lane]": "scratch", "SGPRs Spill": "sgpr_spill",
            "VGPRs Spill": "vgpr_spill", "LDS Size [bytes/block]": "lds", "Occupancy [waves/SIMD]": "occupancy"}
    for m in _REMARK.finditer(text):
        k, v = m.group(1), m.group(2)
        if k == "Function Name":
            cur = out.setdefault(v, {})
        elif cur is not None:
            cur[keys[k]] = int(v)
    return out


def _hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), shutil.which("hipcc"), "/opt/rocm/bin/hipcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("hipcc not found: libs2l_hip.so cannot be built (set HIPCC=...)")


def _older(outputs, sources) -> bool:
    if not all(os.path.exists(o) for o in outputs):
        return True
    t = min(os.path.getmtime(o) for o in outputs)
    return any(os.path.getmtime(d) > t for d in sources)


def _library_needs_build() -> bool:
    return _older([LIB, REF_LIB, RESOURCES], [HEADER] + [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f != TORCH_OPS_SOURCE])


def _torch_ops_need_build() -> bool:
    """_linear_ops.so is missing, older than its sources, or built against another torch."""
    if _older([TORCH_OPS], [HEADER, os.path.join(CSRC, TORCH_OPS_SOURCE)]):
        return True
    import torch
    with open(TORCH_OPS, "rb") as f:
        return f"built for torch {torch.__version__};".encode() not in f.read()


def needs_build() -> bool:
    return _library_needs_build() or _torch_ops_need_build()


def _torch_ops_command() -> list:
    import sysconfig
    import torch
    from torch.utils import cpp_extension
    root = os.path.dirname(torch.__file__)
    include = [os.path.join(root, "include"), os.path.join(root, "include", "torch", "csrc", "api", "include"), sysconfig.get_paths()["include"],
               os.path.join(cpp_extension.ROCM_HOME or "/opt/rocm", "include")]
    return [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            "-DTORCH_API_INCLUDE_EXTENSION_H", f'-DS2L_TORCH_VERSION="{torch.__version__}"', f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *sum((["-isystem", d] for d in include), []),
            os.path.join(CSRC, TORCH_OPS_SOURCE), "-L" + os.path.join(root, "lib"), "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu", "-ltorch_python",
            "-o", TORCH_OPS + ".tmp"]


def build_library(force: bool = False, verbose: bool = False) -> str:
    """Compile every .hip translation unit and link the shared library next to this file; beside it the dense layer's autograd node, without which
    (no g++, no headers of Python or torch) all but autograd.linear works: its failure is a warning."""
    ops = _start_torch_ops() if force or _torch_ops_need_build() else None
    try:
        if force or _library_needs_build():
            _build_hip(verbose)
    finally:
        if ops is not None:
            _finish_torch_ops(ops)
    return LIB


def _start_torch_ops():
    try:
        return subprocess.Popen(_torch_ops_command(), stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    except Exception as e:      # no compiler, no torch to compile against
        return e


def _finish_torch_ops(ops) -> None:
    out = str(ops) if isinstance(ops, Exception) else ops.communicate()[0]
    if not isinstance(ops, Exception) and ops.returncode == 0:
        os.replace(TORCH_OPS + ".tmp", TORCH_OPS)
        return
    if os.path.exists(TORCH_OPS):      # not an old one in its place
        os.remove(TORCH_OPS)
    warnings.warn(f"{TORCH_OPS_SOURCE} was not built, autograd.linear will raise:\n{out}")


def _build_hip(verbose: bool) -> None:
    hipcc = _hipcc()
    objdir = os.path.join(PKG, "build")
    os.makedirs(objdir, exist_ok=True)
    # the renderer's kernel body is generated assembly text (csrc/gen_render_body.py), included by render.hip
    sys.path.insert(0, CSRC)
    try:
        import gen_render_body
        gen_render_body.main_all(objdir)       # render_body.inc (long shape), render_body_wide.inc, render_body_single.inc
        import gen_render_fs_body
        gen_render_fs_body.main(os.path.join(objdir, "render_fs_body.inc"))      # the feature-split tile (one frame per call)
        import gen_rows_fs_body
        gen_rows_fs_body.main(os.path.join(objdir, "rows_fs_body.inc"))          # ... and the general-row MLP's (rgb_forward on a few thousand rows)
        import gen_render16_body
        gen_render16_body.main_all(objdir)     # render16_body_{long,wide,single}.inc: the split-bf16 speed mode (render16.hip)
        import gen_conv16_body
        gen_conv16_body.main(objdir)           # conv16_body.inc: the split-bf16 3x3 convolution of the U-Net's speed mode (conv16.hip)
        import gen_convh_body
        gen_convh_body.main(objdir)            # convh_body.inc: the 3x3 convolution on bf16 tensors of the half-width training chain (convh.hip)
        import gen_convh8_body
        gen_convh8_body.main(objdir)           # convh8_body.inc: its eight-wave form (two waves per SIMD)
        import gen_convhx_body
        gen_convhx_body.main(objdir)           # convhx_body.inc: the eight waves in alternating roles (reference library only; the default is convh8)
        import gen_conv_body               # ... and so are the U-Net's fp32 3x3 convolutions (unet.hip)
        gen_conv_body.main(objdir)
        import gen_fwd16_body              # ... and the bf16 training forward (train_bf16.hip)
        gen_fwd16_body.main(objdir)
        import gen_bwd16_body              # ... and its backward
        gen_bwd16_body.main(objdir)
    finally:
        sys.path.pop(0)
    procs = []
    for src in SOURCES:
        obj = os.path.join(objdir, src.replace(".hip", ".o"))
        cmd = [hipcc, *FLAGS, *SOURCE_FLAGS.get(src, ()), "-I", objdir, "-c", os.path.join(CSRC, src), "-o", obj]
        if verbose:
            print(" ".join(cmd), flush=True)
        procs.append((src, obj, False, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    for src in REF_SOURCES:      # the reference library's own objects, in the same pass
        obj = os.path.join(objdir, "ref_" + src.replace(".hip", ".o"))
        cmd = [hipcc, *FLAGS, "-DS2L_WITH_REFERENCE_KERNELS", "-I", objdir, "-c", os.path.join(CSRC, src), "-o", obj]
        procs.append((src, obj, True, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)))
    objs, ref_objs, resources, ref_resources = [], [], {}, {}
    for src, obj, is_ref, p in procs:
        out, _ = p.communicate()
        if p.returncode != 0:
            raise RuntimeError(f"hipcc failed on {src}{' (reference build)' if is_ref else ''}:\n{out}")
        (ref_resources if is_ref else resources).update(_parse_resources(out))
        rest = "\n".join(l for l in out.splitlines() if "-Rpass-analysis=kernel-resource-usage" not in l and "packed-fp32-ops" not in l)
        if verbose and rest.strip():
            print(rest)
        (ref_objs if is_ref else objs).append(obj)
    ref_names = {s.replace(".hip", ".o") for s in REF_SOURCES}
    for out_lib, parts in ((LIB, objs), (REF_LIB, [o for o in objs if os.path.basename(o) not in ref_names] + ref_objs)):
        cmd = [hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", out_lib + ".tmp", *parts]
        r = subprocess.run(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link of {os.path.basename(out_lib)} failed:\n{r.stdout}")
        os.replace(out_lib + ".tmp", out_lib)
    # per-kernel resources of the product library; the kernels only the reference library holds under "reference_only"
    resources["reference_only"] = {k: v for k, v in ref_resources.items() if k not in resources}
    with open(RESOURCES, "w") as f:
        json.dump(resources, f, indent=0, sort_keys=True)


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose=True))

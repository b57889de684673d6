"""In-tree extension build.

  python setup.py build_ext --inplace

Builds:
  * glint_word2vec_amd._cpu_native     — pybind11 CPU SGNS trainer (always)
  * glint_word2vec_amd._hip_native     — HIP/CDNA4 fused kernels for gfx950
  * glint_word2vec_amd._vocab_native   — HIP/CDNA4 whole-vocabulary kernels
    (whenever hipcc is available; cross-compiles fine without a GPU)

The HIP extensions are compiled by driving hipcc directly (not through
torch.utils.cpp_extension's JIT cache) so the resulting .so lives in-tree
and travels with the repo snapshot to the GPU box.
"""
import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import pybind11
from setuptools import setup, Extension
from setuptools.command.build_ext import build_ext

ROOT = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(ROOT, "glint_word2vec_amd")

cpu_ext = Extension(
    "glint_word2vec_amd._cpu_native",
    sources=["csrc/cpu_sgns.cpp"],
    include_dirs=[pybind11.get_include()],
    extra_compile_args=["-O3", "-std=c++17", "-march=native", "-fvisibility=hidden"],
    language="c++",
)


HIP_EXTENSIONS = {"_hip_native": "sgns_hip.hip",
                  "_vocab_native": "vocab_hip.hip"}


def build_hip_extension(name: str = "_hip_native",
                        force: bool = False) -> str | None:
    """Compile one HIP extension in-tree with hipcc for gfx950.

    Returns the path of the built .so, or None when hipcc is unavailable.
    Deliberately bypasses torch's JIT extension cache: the .so must live
    in-tree so it travels with the repo snapshot to the GPU box.
    """
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        return None
    import sysconfig
    ext_suffix = sysconfig.get_config_var("EXT_SUFFIX") or ".so"
    src = os.path.join(ROOT, "csrc", "hip", HIP_EXTENSIONS[name])
    out = os.path.join(PKG, name + ext_suffix)
    # this file holds the compiler's switches
    needs = (src, os.path.join(ROOT, "setup.py"))
    if not force and os.path.exists(out) and \
            os.path.getmtime(out) > max(map(os.path.getmtime, needs)):
        return out
    cmd = [
        hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC",
        "-shared", "-fvisibility=hidden",
        # packed 32-bit float instructions stay off: scalar code only
        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        "-I", pybind11.get_include(),
        "-I", sysconfig.get_paths()["include"],
        "-x", "hip", src,
        "-o", out,
    ]
    print("building HIP extension:", " ".join(cmd))
    subprocess.check_call(cmd, cwd=ROOT)
    return out


class BuildExt(build_ext):
    def run(self):
        super().run()
        with ThreadPoolExecutor() as pool:      # minutes each
            list(pool.map(lambda name: build_hip_extension(
                name, bool(self.force)), HIP_EXTENSIONS))


setup(
    name="glint_word2vec_amd",
    version="0.1.0",
    packages=["glint_word2vec_amd", "glint_word2vec_amd.models",
              "glint_word2vec_amd.ops", "glint_word2vec_amd.parallel",
              "glint_word2vec_amd.utils"],
    ext_modules=[cpu_ext],
    cmdclass={"build_ext": BuildExt},
)

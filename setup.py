"""In-tree build of the MI355X HIP extension.

    PYTORCH_ROCM_ARCH=gfx950 python setup.py build_ext --inplace

The built elasticdl_amd/ops/_C*.so travels with the repo snapshot to GPU
boxes (it is git-ignored but not gpurun-ignored).
"""

import glob
import hashlib
import os

from setuptools import find_packages, setup

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from torch.utils.cpp_extension import BuildExtension, CUDAExtension  # noqa: E402

ROOT = os.path.dirname(os.path.abspath(__file__))

# ninja follows a source's headers only where the compiler lists them, which
# it does not for HIP: a flag that changes with them makes it compile again
HEADERS = hashlib.sha256()
for header in sorted(glob.glob(
        os.path.join(ROOT, "elasticdl_amd", "ops", "csrc", "*.h"))):
    with open(header, "rb") as f:
        HEADERS.update(f.read())
HEADERS = "-DEDL_HEADERS=0x" + HEADERS.hexdigest()[:16]

ext = CUDAExtension(
    name="elasticdl_amd.ops._C",
    sources=[
        "elasticdl_amd/ops/csrc/bindings.cpp",
        "elasticdl_amd/ops/csrc/ps_kernels.hip",
        "elasticdl_amd/ops/csrc/train_kernels.hip",
        "elasticdl_amd/ops/csrc/gemm_bf16.hip",
        "elasticdl_amd/ops/csrc/bn_kernels.hip",
        "elasticdl_amd/ops/csrc/fp8_bindings.cpp",
        "elasticdl_amd/ops/csrc/fp8_kernels.hip",
        "elasticdl_amd/ops/csrc/embedding_bindings.cpp",
        "elasticdl_amd/ops/csrc/embedding_kernels.hip",
    ],
    extra_compile_args={
        "cxx": ["-O3", "-std=c++17", HEADERS],
        # no packed 32-bit float instructions: some forms of them have given
        # wrong results on this hardware
        "nvcc": ["-O3", "-std=c++17", HEADERS, "-Xclang", "-target-feature",
                 "-Xclang", "-packed-fp32-ops"],
    },
)

setup(
    name="elasticdl_amd",
    version="0.1.0",
    packages=find_packages(include=["elasticdl_amd", "elasticdl_amd.*"]),
    entry_points={
        "console_scripts": ["elasticdl=elasticdl_amd.client.main:main"],
    },
    ext_modules=[ext],
    cmdclass={"build_ext": BuildExtension},
)

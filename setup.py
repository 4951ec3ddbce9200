"""Build the gfx950 native extension IN-TREE.

    PYTORCH_ROCM_ARCH=gfx950 python setup.py build_ext --inplace

The .so lands next to the package (spark_sklearn_amd/_hip_ops*.so) so it
travels with the repo snapshot to the GPU box (no JIT cache dependence).
"""

import glob
import os
import sys

from setuptools import setup

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from torch.utils.cpp_extension import BuildExtension, CUDAExtension  # noqa: E402

HEADERS = ["spark_sklearn_amd/ops/csrc/ska_rows.h"]

# ninja knows nothing of the headers that HIP sources include: objects that
# are older than one of them are built again
newest = max(os.path.getmtime(h) for h in HEADERS)
for built in glob.glob("build/temp*/spark_sklearn_amd/ops/csrc/*.o"):
    if os.path.getmtime(built) < newest:
        os.remove(built)

ext = CUDAExtension(
    name="spark_sklearn_amd._hip_ops",
    sources=["spark_sklearn_amd/ops/csrc/ska_ops.hip",
             "spark_sklearn_amd/ops/csrc/ska_grouped.hip"],
    depends=HEADERS,
    extra_compile_args={
        "cxx": ["-O3", "-std=c++17"],
        # packed fp32 instructions stay off: hipcc makes them from ordinary
        # float code, and some of their forms have given wrong results
        "nvcc": ["-O3", "-std=c++17", "--offload-arch=gfx950",
                 "-Xclang", "-target-feature",
                 "-Xclang", "-packed-fp32-ops"],
    },
)

setup(
    name="spark_sklearn_amd",
    version="0.1.0",
    packages=["spark_sklearn_amd", "spark_sklearn_amd.models",
              "spark_sklearn_amd.ops", "spark_sklearn_amd.parallel"],
    ext_modules=[ext],
    cmdclass={"build_ext": BuildExtension},
)

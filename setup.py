"""Build the in-tree gfx950 HIP extension.

    PYTORCH_ROCM_ARCH=gfx950 python setup.py build_ext --inplace

The .so lands at gradient_accumulation_tf_estimator_amd/ops/_ga_hip*.so so it
travels with repo snapshots to GPU boxes (no JIT cache involved).
"""

import glob
import hashlib
import os

os.environ.setdefault("PYTORCH_ROCM_ARCH", "gfx950")

from setuptools import setup  # noqa: E402
from torch.utils.cpp_extension import BuildExtension, CUDAExtension  # noqa: E402

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "gradient_accumulation_tf_estimator_amd", "ops", "csrc")

# hipcc -O3 turns ordinary float code into the packed FP32 forms
# (v_pk_add/mul/fma_f32); they are kept out of every kernel. The host pass
# does not know the feature and only warns.
NO_PACKED_FP32 = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]

# Objects are rebuilt when their command changes, not when a header does: the
# headers' digest is part of the command.
_digest = hashlib.sha256()
for _h in sorted(glob.glob(os.path.join(CSRC, "*.h"))):
    with open(_h, "rb") as _f:
        _digest.update(_f.read())
HEADERS = ["-DGA_HEADERS=0x" + _digest.hexdigest()[:8]]

setup(
    name="gradient_accumulation_tf_estimator_amd",
    version="0.1.0",
    packages=["gradient_accumulation_tf_estimator_amd"],
    ext_modules=[
        CUDAExtension(
            name="gradient_accumulation_tf_estimator_amd.ops._ga_hip",
            sources=[
                os.path.join(CSRC, "ga_kernels.hip"),
                os.path.join(CSRC, "fused_ln_gelu.hip"),
                os.path.join(CSRC, "blas_acc.hip"),
                os.path.join(CSRC, "lt_gemm.hip"),
                os.path.join(CSRC, "grouped_wgrad.hip"),
                os.path.join(CSRC, "attn.hip"),
                os.path.join(CSRC, "wgrad_mfma.hip"),
                os.path.join(CSRC, "ffn_mfma.hip"),
                os.path.join(CSRC, "cls_head.hip"),
                os.path.join(CSRC, "linear_small.hip"),
                os.path.join(CSRC, "rms_norm.hip"),
                os.path.join(CSRC, "grad_clip.hip"),
                os.path.join(CSRC, "rel_attn.hip"),
                os.path.join(CSRC, "ops_bindings.hip"),
                os.path.join(CSRC, "ga_bindings.hip"),
            ],
            libraries=["hipblaslt"],
            # GA_ASAN=1: instrument the HOST side (bindings, launch plumbing,
            # hipBLASLt workspace management) with AddressSanitizer; device
            # code is unchanged. Run via tools/asan_smoke.sh (LD_PRELOADs
            # libasan). Device-side ASAN needs xnack+ and is not exercised
            # on this pool.
            # Compile-only instrumentation: the __asan_* references stay
            # undefined in the .so (legal for shared objects) and resolve
            # from the LD_PRELOADed clang runtime at run time -- the link
            # step is g++, whose libasan must not be mixed in.
            extra_compile_args={
                "cxx": ["-O3"] + (["-fsanitize=address", "-g"]
                                  if os.environ.get("GA_ASAN") else []),
                "nvcc": ["-O3", "--offload-arch=gfx950"] + NO_PACKED_FP32 + HEADERS
                + (["-fsanitize=address", "-g",
                    "-Xarch_device", "-fno-sanitize=all"]
                   if os.environ.get("GA_ASAN") else []),
            },
        )
    ],
    cmdclass={"build_ext": BuildExtension},
)

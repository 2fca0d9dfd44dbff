"""In-tree build of the gfx950 HIP extensions.

Usage:  PYTORCH_ROCM_ARCH=gfx950 python setup.py build_ext --inplace

Builds:
  mgwfbp_amd/kernels/mgx_kernels_ext*.so   (fused SGD / pack / unpack / norm)
  mgwfbp_amd/kernels/mgx_bn_ext*.so        (NHWC BatchNorm and max pooling)
  mgwfbp_amd/kernels/mgx_lm_ext*.so        (language-model operators)
  mgwfbp_amd/comm/mgx_comm_ext*.so         (RCCL comm core)

The .so files are git-ignored but travel with the gpurun snapshot, so a
CPU-side cross-compile here runs unchanged on the MI355X box.
"""
import os

from setuptools import setup

os.environ.setdefault('PYTORCH_ROCM_ARCH', 'gfx950')

from torch.utils.cpp_extension import BuildExtension, CUDAExtension  # noqa: E402

ROOT = os.path.dirname(os.path.abspath(__file__))

# Device code is built without packed fp32 arithmetic: hipcc -O3 forms
# v_pk_{add,mul,fma}_f32 from ordinary float code by itself, and some of
# their forms have given wrong results on gfx950. Nearly all kernels here
# are bound by memory, and the scalar forms cost them nothing that shows:
# ResNet-50's BatchNorm backward sums took 37.7 us with the packed forms and
# take 37.4 without, its other passes 65.3 and 66.5, 41.6 and 43.5, while
# the libraries' convolutions beside them, the same code, took 2 to 9% more
# in the second run. (hipcc's host pass warns that it does not know the
# feature; that is harmless.)
common_args = {
    'cxx': ['-O3', '-std=c++17'],
    'nvcc': ['-O3', '-std=c++17', '-Xclang', '-target-feature',
             '-Xclang', '-packed-fp32-ops'],
}

ext_modules = [
    CUDAExtension(
        name='mgwfbp_amd.kernels.mgx_kernels_ext',
        sources=['mgwfbp_amd/kernels/mgx_kernels.hip'],
        extra_compile_args=common_args,
    ),
    CUDAExtension(
        name='mgwfbp_amd.kernels.mgx_bn_ext',
        sources=['mgwfbp_amd/kernels/bn_kernels.hip'],
        extra_compile_args=common_args,
    ),
    CUDAExtension(
        name='mgwfbp_amd.kernels.mgx_lm_ext',
        sources=['mgwfbp_amd/kernels/lm_ext.hip',
                 'mgwfbp_amd/kernels/embedding_kernels.hip',
                 'mgwfbp_amd/kernels/grad_clip_kernels.hip',
                 'mgwfbp_amd/kernels/token_loss_kernels.hip'],
        depends=['mgwfbp_amd/kernels/lm_common.h'],
        extra_compile_args=common_args,
    ),
    CUDAExtension(
        name='mgwfbp_amd.comm.mgx_comm_ext',
        sources=['mgwfbp_amd/comm/comm_core.hip'],
        libraries=['rccl'],
        extra_compile_args=common_args,
    ),
]

setup(
    name='mgwfbp_amd',
    version='0.1.0',
    description='MI355X-native merged-gradient WFBP training framework',
    packages=['mgwfbp_amd', 'mgwfbp_amd.comm', 'mgwfbp_amd.kernels',
              'mgwfbp_amd.models', 'mgwfbp_amd.data'],
    ext_modules=ext_modules,
    cmdclass={'build_ext': BuildExtension},
)

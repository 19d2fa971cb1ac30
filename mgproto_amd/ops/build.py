"""Build the in-tree mgproto_hip extension for gfx950.

Usage: ``python -m mgproto_amd.ops.build``. Cross-compiles on CPU-only boxes
(hipcc needs no GPU); the resulting ``_mgproto_hip.so`` sits in-tree so it
travels with repo snapshots.
"""

import glob
import os
import shutil
import sys

_HERE = os.path.dirname(os.path.abspath(__file__))
SRC = [os.path.join(_HERE, 'hip', 'mgproto_kernels.hip'),
       os.path.join(_HERE, 'hip', 'fused_bn.hip'),
       os.path.join(_HERE, 'hip', 'em_kernels.hip'),
       os.path.join(_HERE, 'hip', 'enqueue_kernels.hip'),
       os.path.join(_HERE, 'hip', 'gemm1x1_kernels.hip'),
       os.path.join(_HERE, 'hip', 'mx4_quant.hip'),
       os.path.join(_HERE, 'hip', 'mx4_linear.hip'),
       os.path.join(_HERE, 'hip', 'mx4_tiles.hip'),
       os.path.join(_HERE, 'hip', 'mx4_rounding.hip'),
       os.path.join(_HERE, 'hip', 'mx4_grad.hip'),
       os.path.join(_HERE, 'hip', 'mx4_grad_input.hip'),
       os.path.join(_HERE, 'hip', 'mx4_grad_weight.hip'),
       os.path.join(_HERE, 'hip', 'grad_clip.hip'),
       os.path.join(_HERE, 'hip', 'mx4_bindings.hip'),
       os.path.join(_HERE, 'hip', 'graph_fill.hip')]
# no packed fp32 instructions: some of their forms give wrong results on this
# hardware now and then (hipcc's host pass warns that it has no such feature)
HIP_FLAGS = ['-O3', '-Xclang', '-target-feature', '-Xclang',
             '-packed-fp32-ops']
OUT = os.path.join(_HERE, '_mgproto_hip.so')
CPU_SRC = [os.path.join(_HERE, 'cpu', 'fastaug.cpp')]
CPU_OUT = os.path.join(_HERE, '_mgproto_cpu.so')


def build_cpu(verbose: bool = False) -> str:
    """Native CPU augmentation core (plain C++, OpenMP via at::parallel)."""
    from torch.utils.cpp_extension import load
    build_dir = os.path.join(_HERE, 'cpu', 'build')
    os.makedirs(build_dir, exist_ok=True)
    load(name='_mgproto_cpu', sources=CPU_SRC, build_directory=build_dir,
         extra_cflags=['-O3', '-fopenmp'], verbose=verbose,
         is_python_module=True)
    built = os.path.join(build_dir, '_mgproto_cpu.so')
    if os.path.isfile(built):
        shutil.copy2(built, CPU_OUT)
    return CPU_OUT


def _drop_stale(build_dir: str):
    """Objects older than a header: the generated ninja file knows only their
    sources."""
    newest = max((os.path.getmtime(h) for h in
                  glob.glob(os.path.join(_HERE, 'hip', '*.h'))), default=0)
    for src in SRC:
        with open(src) as f:
            local = '#include "' in f.read()
        obj = os.path.join(build_dir, os.path.basename(src)[:-4] + '.cuda.o')
        if local and os.path.isfile(obj) and os.path.getmtime(obj) < newest:
            os.remove(obj)


def build(verbose: bool = False) -> str:
    os.environ.setdefault('PYTORCH_ROCM_ARCH', 'gfx950')
    os.environ.setdefault('MAX_JOBS', '8')
    from torch.utils.cpp_extension import load

    build_dir = os.path.join(_HERE, 'hip', 'build')
    os.makedirs(build_dir, exist_ok=True)
    _drop_stale(build_dir)
    mod = load(name='_mgproto_hip',
               sources=SRC,
               build_directory=build_dir,
               extra_cflags=['-O3'],
               extra_cuda_cflags=HIP_FLAGS,
               verbose=verbose,
               is_python_module=True)
    built = os.path.join(build_dir, '_mgproto_hip.so')
    if os.path.isfile(built):
        shutil.copy2(built, OUT)
    return OUT


if __name__ == '__main__':
    path = build(verbose='-v' in sys.argv)
    print(f'built {path}')
    path = build_cpu(verbose='-v' in sys.argv)
    print(f'built {path}')

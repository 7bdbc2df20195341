"""Builds libfiery_hip.so (gfx950) in-tree with hipcc, and _row_autograd.so - the row operators' autograd nodes, host C++ against
PyTorch's headers - with g++.  `python -m fiery_amd.build [--force]`."""
import os
import subprocess
import sys
import sysconfig

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
INCLUDE = os.path.join(os.path.dirname(HERE), 'include')
OUT = os.path.join(HERE, 'libfiery_hip.so')
HIPCC = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')

# (source, extra flags).  lift_splat.hip: the index path must round like ATen's CPU kernels -> no FMA contraction.
SOURCES = [
    ('runtime.cpp', []),
    ('lift_splat.hip', ['-ffp-contract=off']),
    ('warp.hip', ['-ffp-contract=off']),                # sampling positions round like ATen's CPU kernels (see the file)
    ('conv_igemm.hip', []),
    # one translation unit per tile shape of the convolution kernel: they compile side by side
    ('conv_tile_128x32.hip', []),
    ('conv_tile_128x64.hip', []),
    ('conv_tile_128x128.hip', []),
    ('conv_tile_128x128_rest.hip', []),
    ('conv_tile_64x64.hip', []),
    ('conv_tile_64x128.hip', []),
    ('conv_tile_bf16_a.hip', []),
    ('conv_tile_bf16_b.hip', []),
    ('conv_tile_halo_f32.hip', []),
    ('conv_tile_stream_k.hip', []),
    ('conv_tile_split.hip', []),
    ('conv_winograd.hip', []),
    ('conv_winograd_split.hip', []),
    ('aux_ops.hip', []),
    ('conv_grad.hip', []),
    ('bn_train.hip', []),
    ('gru_train.hip', []),
    ('layer_norm.hip', []),
    ('dropout.hip', []),
    ('dropout_norm.hip', []),
    ('labels.hip', []),
    ('images.hip', []),
]
# FIERY_CONV_TUNING=1: also build the convolution's clock-probe / priority variants (tools/microbench.py conv --clk)
TUNING = ['-DFIERY_CONV_TUNING=1'] if os.environ.get('FIERY_CONV_TUNING') == '1' else ['-DFIERY_CONV_TUNING=0']
# hipcc turns plain float code into packed fp32 instructions by itself; these translation units are built without them (a device
# feature: hipcc's host pass warns that it does not know it)
NO_PACKED_FP32 = ['-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
HIP_ONLY = {name: NO_PACKED_FP32 for name in ('layer_norm.hip', 'dropout.hip', 'dropout_norm.hip')}
COMMON = ['--offload-arch=gfx950', '-O3', '-std=c++17', '-fPIC', '-I' + INCLUDE, '-I' + CSRC, '-x', 'hip']


# the row operators' autograd nodes (host code; reaches the library through addresses, so it links against PyTorch only)
AUTOGRAD_SOURCE = os.path.join(CSRC, 'row_autograd.cpp')
AUTOGRAD_OUT = os.path.join(HERE, '_row_autograd.so')


def _autograd_command():
    import torch
    base = os.path.dirname(torch.__file__)
    return [os.environ.get('CXX', 'g++'), '-O2', '-std=c++17', '-fPIC', '-shared', '-fvisibility=hidden', f'-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}',
            '-I' + INCLUDE, f'-I{base}/include', f'-I{base}/include/torch/csrc/api/include', '-I' + sysconfig.get_paths()['include'], AUTOGRAD_SOURCE,
            '-o', AUTOGRAD_OUT, f'-L{base}/lib', '-ltorch_python', '-ltorch_cpu', '-ltorch', '-lc10']


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=True):
    # FIERY_BUILD_VARIANT=name (+ FIERY_BUILD_FLAGS="-D..."): a second library for A/B runs on one GPU box,
    # tools/ab/libfiery_hip_<name>.so, selected with FIERY_HIP_LIB=...; the in-tree library is left alone
    variant = os.environ.get('FIERY_BUILD_VARIANT')
    global OUT
    objdir = os.path.join(HERE, 'build' if not variant else 'build_' + variant)
    if variant:
        os.makedirs(os.path.join(os.path.dirname(HERE), 'tools', 'ab'), exist_ok=True)
        OUT = os.path.join(os.path.dirname(HERE), 'tools', 'ab', f'libfiery_hip_{variant}.so')
    os.makedirs(objdir, exist_ok=True)
    headers = [os.path.join(CSRC, 'common.h'), os.path.join(CSRC, 'conv_igemm_kernel.h'),
               os.path.join(CSRC, 'fiery_gfx950.h'), os.path.join(CSRC, 'fiery_row_types.h'), os.path.join(CSRC, 'row_ops.h'),
               os.path.join(CSRC, 'layer_norm_kernel.h'), os.path.join(INCLUDE, 'fiery_hip.h')]
    objs, jobs = [], []
    for name, extra in SOURCES:
        src = os.path.join(CSRC, name)
        obj = os.path.join(objdir, name + '.o')
        objs.append(obj)
        if force or _stale(obj, [src] + headers):
            cmd = [HIPCC] + COMMON + TUNING + os.environ.get('FIERY_BUILD_FLAGS', '').split() + extra + HIP_ONLY.get(name, []) + ['-c', src, '-o', obj]
            if verbose:
                print(' '.join(cmd), flush=True)
            jobs.append((name, subprocess.Popen(cmd)))       # translation units compile side by side
    if not variant and (force or _stale(AUTOGRAD_OUT, [AUTOGRAD_SOURCE, os.path.join(INCLUDE, 'fiery_hip.h')])):
        cmd = _autograd_command()
        if verbose:
            print(' '.join(cmd), flush=True)
        jobs.append(('row_autograd.cpp', subprocess.Popen(cmd)))
    failed = [name for name, proc in jobs if proc.wait() != 0]
    if failed:
        raise RuntimeError('hipcc failed for ' + ', '.join(failed))
    if force or _stale(OUT, objs):
        cmd = [HIPCC, '--offload-arch=gfx950', '-shared', '-fPIC', '-o', OUT] + objs
        if verbose:
            print(' '.join(cmd), flush=True)
        subprocess.check_call(cmd)
    return OUT


if __name__ == '__main__':
    build(force='--force' in sys.argv)

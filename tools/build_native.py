"""Build the in-tree HIP extension ``distributed_kfac_pytorch_amd/_C*.so``.

Drives ``hipcc --offload-arch=gfx950`` directly (no hipify, no JIT cache):
every ``csrc/*.hip`` kernel file is compiled to an object, the
``csrc/*.cpp`` host files (bindings, rocSOLVER tier -- the only torch-aware
translation units) are compiled against the installed PyTorch-ROCm headers,
and everything is linked into one shared object next to the Python package
so it travels with the repo snapshot to the GPU box.

Usage:  python tools/build_native.py [--force] [--jobs N] [--verbose]
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import subprocess
import sys
import sysconfig

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, 'csrc')
PKG = os.path.join(ROOT, 'distributed_kfac_pytorch_amd')
BUILD = os.path.join(ROOT, 'build', 'native')
ARCH = os.environ.get('KFAC_OFFLOAD_ARCH', 'gfx950')

# Compiled without packed fp32 instructions (v_pk_add / mul / fma_f32), whose
# results on this card cannot be relied on.  The older kernels keep the flags
# that their results were established with: without packed instructions the
# compiler contracts other products into fma's, and it drops a ReLU mask's
# select in csrc/bnact.hip (20 cases of tests/test_bnact_gpu.py fail).
NO_PACKED_FP32 = ('distill.hip', 'rotary.hip', 'window_attn.hip')
NO_PACKED_FLAGS = ['-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']

# Matrix results that the vector unit reads next stay in vector registers.  By
# default a kernel of more than 256 registers keeps all of them in the
# accumulation half and copies each out before its use (key gradients, heads
# of 128: 124 copies a tile; fp32 there spills 27 registers, and none with it).
MATRIX_IN_VGPRS = ('window_attn.hip',)
MATRIX_IN_VGPRS_FLAGS = ['-mllvm', '-amdgpu-mfma-vgpr-form=1']


def _hipcc() -> str:
    rocm = os.environ.get('ROCM_PATH', '/opt/rocm')
    return os.path.join(rocm, 'bin', 'hipcc')


def _torch_paths() -> tuple[list[str], list[str], bool]:
    import torch
    from torch.utils import cpp_extension

    incs = cpp_extension.include_paths(device_type='cuda')
    libdir = os.path.join(os.path.dirname(torch.__file__), 'lib')
    abi = bool(torch._C._GLIBCXX_USE_CXX11_ABI)
    return incs, [libdir], abi


def ext_suffix() -> str:
    return sysconfig.get_config_var('EXT_SUFFIX') or '.so'


def target_path() -> str:
    return os.path.join(PKG, '_C' + ext_suffix())


def _newer(src_files: list[str], out: str) -> bool:
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(s) > t for s in src_files)


def _other_command(cmd: list[str], obj: str) -> bool:
    """Whether ``obj`` was compiled by another command than ``cmd``."""
    try:
        with open(obj + '.cmd', encoding='utf-8') as f:
            return f.read() != ' '.join(cmd)
    except OSError:
        return True


def _compile(cmd: list[str], obj: str, verbose: bool) -> None:
    _run(cmd, verbose)
    with open(obj + '.cmd', 'w', encoding='utf-8') as f:
        f.write(' '.join(cmd))


def _run(cmd: list[str], verbose: bool) -> None:
    if verbose:
        print(' '.join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError(f'command failed: {" ".join(cmd[:3])} ...')
    if verbose and (r.stdout or r.stderr):
        sys.stderr.write(r.stdout + r.stderr)


def build(force: bool = False, jobs: int = 8, verbose: bool = False) -> str:
    os.makedirs(BUILD, exist_ok=True)
    hipcc = _hipcc()
    incs, libdirs, abi = _torch_paths()
    header_deps = [
        os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.h')
    ]
    common = [
        f'--offload-arch={ARCH}',
        '-O3',
        '-fPIC',
        '-std=c++17',
        '-D__HIP_PLATFORM_AMD__=1',
        '-DUSE_ROCM=1',
        f'-D_GLIBCXX_USE_CXX11_ABI={int(abi)}',
        f'-I{CSRC}',
    ]
    kernel_srcs = sorted(
        os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.hip')
    )
    jobs_list = []
    objs = []
    for src in kernel_srcs:
        obj = os.path.join(BUILD, os.path.basename(src) + '.o')
        objs.append(obj)
        extra = NO_PACKED_FLAGS if os.path.basename(src) in NO_PACKED_FP32 else []
        if os.path.basename(src) in MATRIX_IN_VGPRS:
            extra = extra + MATRIX_IN_VGPRS_FLAGS
        cmd = [hipcc, *common, *extra, '-c', src, '-o', obj]
        if force or _newer([src] + header_deps, obj) or _other_command(cmd, obj):
            jobs_list.append((cmd, obj))
    py_inc = sysconfig.get_paths()['include']
    torch_srcs = sorted(
        os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.cpp')
    )
    for src in torch_srcs:
        obj = os.path.join(BUILD, os.path.basename(src) + '.o')
        objs.append(obj)
        cmd = [
            hipcc,
            *common,
            '-DTORCH_EXTENSION_NAME=_C',
            '-DTORCH_API_INCLUDE_EXTENSION_H',
            '-Wno-unused-result',
            '-Wno-deprecated-declarations',
            *[f'-I{p}' for p in incs],
            f'-I{py_inc}',
            '-c',
            src,
            '-o',
            obj,
        ]
        if force or _newer([src] + header_deps, obj) or _other_command(cmd, obj):
            jobs_list.append((cmd, obj))
    with cf.ThreadPoolExecutor(max_workers=max(1, jobs)) as ex:
        futs = [ex.submit(_compile, cmd, obj, verbose) for cmd, obj in jobs_list]
        for f in futs:
            f.result()
    out = target_path()
    if force or jobs_list or not os.path.exists(out):
        link = [
            hipcc,
            f'--offload-arch={ARCH}',
            '-shared',
            '-fPIC',
            *objs,
            '-o',
            out,
            *[f'-L{d}' for d in libdirs],
            *[f'-Wl,-rpath,{d}' for d in libdirs],
            '-lc10',
            '-lc10_hip',
            '-ltorch',
            '-ltorch_cpu',
            '-ltorch_hip',
            '-ltorch_python',
            '-lamdhip64',
            '-L/opt/rocm/lib',
            '-Wl,-rpath,/opt/rocm/lib',
            '-lrocsolver',
            '-lrocblas',
        ]
        _run(link, verbose)
    return out


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument('--force', action='store_true')
    ap.add_argument('--jobs', type=int, default=min(8, os.cpu_count() or 1))
    ap.add_argument('--verbose', action='store_true')
    args = ap.parse_args()
    print(build(args.force, args.jobs, args.verbose))


if __name__ == '__main__':
    main()

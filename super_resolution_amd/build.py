"""Builds libsr_amd.so in-tree with hipcc for gfx950 (cross-compiles without a GPU).

    python -m super_resolution_amd.build [--force]
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
SOURCES = ['layout.hip', 'fbm.hip', 'fbm_fast.hip', 'fbm_fast_mixed.hip', 'fbm_mfma.hip', 'gates.hip', 'weightgen.hip', 'weightgen_bwd.hip', 'conv.hip', 'conv_plain.hip', 'net.hip', 'head.hip', 'train.hip', 'adamw.hip']
# no packed float32 instructions: some of their forms have given wrong results on gfx950 now and then
# (measured on a batch of 16 512x512 images, 692.9 and 694.0 ms with them, 692.7 and 693.4 without, and on the training step; the tiled,
# plain and SRVGG workloads were not compared)
FLAGS = ['-O3', '--offload-arch=gfx950', '-std=c++17', '-fno-signed-zeros', '-fPIC', '-Wall', '-Wno-unused-result', '-Xclang', '-target-feature', '-Xclang',
         '-packed-fp32-ops']
# adamw.hip: every operation rounded once (its results are those of the formulas, bit for bit)
EXTRA = {'adamw.hip': ['-ffp-contract=off']}
OUT = os.path.join(HERE, 'libsr_amd.so')
HOST_SRC = os.path.join(CSRC, 'torch_host.cpp')
HOST_OUT = os.path.join(HERE, 'libsr_amd_torch.so')


def _stale():
    if not os.path.exists(OUT):
        return True
    t = os.path.getmtime(OUT)
    deps = [os.path.join(CSRC, f) for f in os.listdir(CSRC)] + [os.path.join(HERE, '..', 'include', 'sr_amd.h')]
    return any(os.path.getmtime(d) > t for d in deps)


def _host_command():
    """g++ line of the small library that reads torch's tensor objects (csrc/torch_host.cpp)."""
    import sysconfig
    import torch
    root = os.path.dirname(torch.__file__)
    # -O3: the walk over 8380 tensors takes 71 us, 84 with -O2
    return ['g++', '-O3', '-std=c++17', '-fPIC', '-shared', '-Wall', '-fvisibility=hidden', '-D_GLIBCXX_USE_CXX11_ABI=%d' % torch.compiled_with_cxx11_abi(),
            '-isystem', os.path.join(root, 'include'), '-isystem', os.path.join(root, 'include', 'torch', 'csrc', 'api', 'include'),
            '-isystem', sysconfig.get_paths()['include'], HOST_SRC, '-o', HOST_OUT,
            '-L' + os.path.join(root, 'lib'), '-ltorch_python', '-ltorch_cpu', '-lc10']


def build(force=False, verbose=True):
    host = None
    if force or not os.path.exists(HOST_OUT) or os.path.getmtime(HOST_SRC) > os.path.getmtime(HOST_OUT):
        cmd = _host_command()
        host = (cmd, subprocess.Popen(cmd))
    try:
        if force or _stale():
            _build_kernels(force, verbose)
    finally:
        if host and host[1].wait() != 0:
            raise RuntimeError('g++ failed: ' + ' '.join(host[0]))
    return OUT


def _build_kernels(force, verbose):
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
    objs = []
    procs = []
    os.makedirs(os.path.join(HERE, 'build'), exist_ok=True)
    headers = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith('.h')] + [os.path.join(HERE, '..', 'include', 'sr_amd.h')]
    newest_header = max(os.path.getmtime(h) for h in headers)
    for s in SOURCES:
        o = os.path.join(HERE, 'build', s.replace('.hip', '.o'))
        objs.append(o)
        src = os.path.join(CSRC, s)
        if not force and os.path.exists(o) and os.path.getmtime(o) > max(os.path.getmtime(src), newest_header):
            continue  # object is newer than its source and every header
        cmd = [hipcc] + FLAGS + EXTRA.get(s, []) + ['-c', os.path.join(CSRC, s), '-o', o]
        procs.append((cmd, subprocess.Popen(cmd)))
    for cmd, p in procs:
        if p.wait() != 0:
            raise RuntimeError('hipcc failed: ' + ' '.join(cmd))
    cmd = [hipcc, '--offload-arch=gfx950', '-shared', '-fPIC'] + objs + ['-o', OUT]
    subprocess.check_call(cmd)
    if verbose:
        print('built', OUT)


if __name__ == '__main__':
    build(force='--force' in sys.argv)

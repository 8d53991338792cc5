"""Build libadvmix_hip.so (gfx950 only) with hipcc, and the torch-side module _node.so.  `python -m advmix_amd.build`."""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, 'csrc')
SO = os.path.join(HERE, 'libadvmix_hip.so')
SOURCES = ['conv_mfma.hip', 'conv_direct.hip', 'conv_wino.hip', 'conv_wino4.hip', 'conv_smap.hip', 'conv_pw.hip', 'wgrad_direct.hip', 'wgrad_lds.hip', 'wgrad_wino.hip', 'norm.hip', 'layer_norm.hip', 'pointwise.hip', 'advmix_ops.hip', 'adamw.hip', 'postproc.hip', 'inputpipe.hip', 'nms.hip']
FLAGS = ['-O3', '--offload-arch=gfx950', '-fPIC', '-munsafe-fp-atomics', '-std=c++17',
         '-Wno-unused-result', '-Wno-pass-failed',     # (pass-failed: 'occupancy target not met' where LDS, not registers, is the limit)
         # No packed fp32 instructions (v_pk_fma_f32 and its like): the compiler makes them of ordinary float code, and some
         # of their forms have given wrong results now and then.  (hipcc's host pass says that it does not know the feature.)
         '-Xclang', '-target-feature', '-Xclang', '-packed-fp32-ops']
# Every kernel must fit its registers: a kernel with scratch (spilled VGPRs) is refused - none of the library's kernels needs
# any, a spill is always an accident of a register cap, and spilling builds were among the suspects of round 3's
# two-process NaN hunt (conv_direct.hip, at its launch bounds).  The compiler reports each kernel's scratch; the build reads it.
RESOURCE_FLAG = '-Rpass-analysis=kernel-resource-usage'


# The layer norm's autograd node: host code against torch's headers, a module of its own (the library knows no torch types).
NODE, NODE_SO = 'layer_norm_node.cpp', os.path.join(HERE, '_node.so')


def _node_command():
    import sysconfig
    import torch
    inc = os.path.join(os.path.dirname(torch.__file__), 'include')
    lib = os.path.join(os.path.dirname(torch.__file__), 'lib')
    rocm = os.environ.get('ROCM_PATH', '/opt/rocm')
    return [os.environ.get('CXX', 'g++'), '-O2', '-std=c++17', '-fPIC', '-shared', '-D__HIP_PLATFORM_AMD__=1', '-DUSE_ROCM=1',
            '-D_GLIBCXX_USE_CXX11_ABI=%d' % torch.compiled_with_cxx11_abi(), '-I' + inc, '-I' + os.path.join(inc, 'torch/csrc/api/include'),
            '-I' + os.path.join(rocm, 'include'), '-I' + sysconfig.get_paths()['include'], os.path.join(CSRC, NODE), '-o', NODE_SO,
            '-L' + lib, '-L' + os.path.join(rocm, 'lib'), '-ltorch_python', '-ltorch_cpu', '-ltorch', '-lc10', '-lc10_hip', '-lamdhip64', '-DADVMIX_TORCH="%s"' % torch.__version__]


def _scratch_users(report):
    """Kernels with scratch in a -Rpass-analysis=kernel-resource-usage report: [(function, bytes per lane)]."""
    import re
    out, name = [], None
    for line in report.splitlines():
        m = re.search(r'remark: Function Name: (\S+)', line)
        if m:
            name = m.group(1)
            continue
        m = re.search(r'ScratchSize \[bytes/lane\]: (\d+)', line)
        if m and int(m.group(1)) > 0:
            out.append((name, int(m.group(1))))
    return out


def _sha(path):
    import hashlib
    with open(path, 'rb') as f:
        return hashlib.sha256(f.read()).hexdigest()[:16]


def _stale(out, deps):
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(d) > t for d in deps)


def _load_info():
    import json
    try:
        with open(os.path.join(HERE, 'build_info.json')) as f:
            return json.load(f)
    except (OSError, ValueError):
        return {'objects': {}}


def _stale_object(s, obj, src, hdrs, info):
    """Does ``obj`` have to be recompiled?  By CONTENT where build_info.json knows what the object was compiled from (the
    source's and the headers' hashes at that time: a checkout that sets mtimes its own way must neither
    rebuild everything nor - worse - keep an object of an older source), by mtime otherwise."""
    if not os.path.exists(obj):
        return True
    rec = info.get('objects', {}).get(s)
    if rec and rec.get('headers_sha256_16') is not None and rec.get('flags') is not None:
        return (rec.get('source_sha256_16') != _sha(src) or rec['headers_sha256_16'] != {os.path.basename(h): _sha(h) for h in hdrs}
                or rec['flags'] != (_node_command() if s == NODE else FLAGS))
    return _stale(obj, [src] + hdrs)


def build(force=False, verbose=True):
    hipcc = os.environ.get('HIPCC', '/opt/rocm/bin/hipcc')
    hdrs = [os.path.join(CSRC, 'common.h'), os.path.join(HERE, '..', 'include', 'advmix_hip.h')]
    objs = []
    procs = []
    info = _load_info()
    for s in SOURCES:
        src = os.path.join(CSRC, s)
        obj = os.path.join(CSRC, s.replace('.hip', '.o'))
        objs.append(obj)
        if force or _stale_object(s, obj, src, hdrs, info):
            cmd = [hipcc] + FLAGS + [RESOURCE_FLAG, '-c', src, '-o', obj]
            if verbose:
                print(' '.join(cmd), flush=True)
            procs.append((s, obj, subprocess.Popen(cmd, stderr=subprocess.PIPE, text=True)))
    node_error = None                                       # (told when the library is there: only one op needs the module)
    if force or _stale_object(NODE, NODE_SO, os.path.join(CSRC, NODE), [], info):
        cmd = _node_command()
        if verbose:
            print(' '.join(cmd), flush=True)
        try:
            procs.append((NODE, NODE_SO, subprocess.Popen(cmd, stderr=subprocess.PIPE, text=True)))
        except OSError as e:
            node_error = str(e)
    bad = []
    for s, obj, p in procs:
        _, err = p.communicate()
        other = [ln for ln in err.splitlines() if 'kernel-resource-usage' not in ln]
        # (the remark lines carry a source excerpt each: print only what is not part of the resource report)
        msgs = [ln for ln in other if ('warning' in ln or 'error' in ln) and 'packed-fp32-ops' not in ln]
        if msgs and verbose:
            print('\n'.join(msgs), flush=True)
        if p.returncode != 0:
            sys.stderr.write(err[-4000:])
            if s != NODE:
                raise RuntimeError('hipcc failed on ' + s)
            node_error = 'the C++ compiler failed'
        users = _scratch_users(err)
        if users:
            os.remove(obj)                                  # never link it
            bad += ['%s: %s uses %d bytes of scratch per lane' % (s, n, b) for n, b in users]
    if bad:
        _record(hipcc, [s for s, obj, _ in procs if os.path.exists(obj)], False)      # what DID compile stays recorded
        raise RuntimeError('kernels with register spills / scratch are refused (see build.py):\n  ' + '\n  '.join(bad))
    linked = False
    if force or any(s != NODE for s, _, _ in procs) or _stale(SO, objs):
        cmd = [hipcc, '--offload-arch=gfx950', '-shared', '-fPIC', '-o', SO] + objs
        if verbose:
            print(' '.join(cmd), flush=True)
        subprocess.check_call(cmd)
        linked = True
    _record(hipcc, [s for s, _, _ in procs if s != NODE or node_error is None], linked)
    if node_error is not None:
        raise RuntimeError('%s on %s (the library itself is built)' % (node_error, NODE))
    return SO


def _record(hipcc, compiled, linked):
    """advmix_amd/build_info.json: what THIS call compiled / linked and what the library on disk was built from (source
    hashes at build time), so that a reader of the tree can tell whether the .so the tests loaded matches the sources
    next to it (build(force=False) reuses objects by mtime and nothing recorded it)."""
    import hashlib
    import json
    import time

    def sha(path):
        with open(path, 'rb') as f:
            return hashlib.sha256(f.read()).hexdigest()[:16]
    info_path = os.path.join(HERE, 'build_info.json')
    try:
        with open(info_path) as f:
            info = json.load(f)
    except (OSError, ValueError):
        info = {'objects': {}}
    hdrs = {h: sha(os.path.join(HERE, *h.split('/'))) for h in ('csrc/common.h', '../include/advmix_hip.h')}
    for s in compiled:
        info['objects'][s] = {'source_sha256_16': sha(os.path.join(CSRC, s)), 'compiled_at': time.strftime('%Y-%m-%d %H:%M:%S'),
                              'headers_sha256_16': {} if s == NODE else {os.path.basename(h): v for h, v in hdrs.items()},
                              'flags': _node_command() if s == NODE else FLAGS}
    info.update({'last_call': {'at': time.strftime('%Y-%m-%d %H:%M:%S'), 'compiled': compiled, 'linked': linked},
                 'headers_sha256_16': hdrs, 'flags': FLAGS,
                 'sources_now': {s: sha(os.path.join(CSRC, s)) for s in SOURCES + [NODE]},
                 'library_sha256_16': sha(SO) if os.path.exists(SO) else None})
    info['up_to_date'] = all(info['objects'].get(s, {}).get('source_sha256_16') == h for s, h in info['sources_now'].items())
    try:
        info['hipcc'] = subprocess.run([hipcc, '--version'], capture_output=True, text=True).stdout.strip().splitlines()[0]
    except OSError:
        pass
    with open(info_path, 'w') as f:
        json.dump(info, f, indent=1, sort_keys=True)
    return info


if __name__ == '__main__':
    build(force='--force' in sys.argv)

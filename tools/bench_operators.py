#!/usr/bin/env python3
"""Times of the layer norm and of AdamW: the source of the figures beside the kernels and in the table of cases.

usage: bench_operators.py                 the rates of this card (a large copy, large matrix products); then each case of
                                          perf/operators.py: an eager pass (host and GPU, one after another) and the same passes
                                          replayed from a HIP graph (the GPU alone)
       bench_operators.py --kernels       single kernels, replayed from a HIP graph, at the sizes that the kernels' comments name
       bench_operators.py --passes N      N eager passes of each case, for a profiler
       bench_operators.py --table DIR     kernel table (CSV) from DIR/{time,fetch,write}_*.csv of profiled runs of --passes

Three sets of data take turns everywhere, each with outputs of its own, so that large cases come from memory and small ones from
the caches.  tools/profile_operators.sh runs all of it."""
import csv
import glob
import importlib.util
import os
import re
import statistics
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
SETS, OURS = 3, ('ln_', 'adamw', 'sumsq', 'tick')


def cases():
    spec = importlib.util.spec_from_file_location('operators', os.path.join(ROOT, 'perf', 'operators.py'))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.own = True
    return m


def wall(f, n):
    import torch
    for _ in range(3):
        f()
    torch.cuda.synchronize()
    a = time.perf_counter()
    for _ in range(n):
        f()
    torch.cuda.synchronize()
    return (time.perf_counter() - a) / n * 1e6


def graph_us(calls, reps=6):
    """Microseconds of one of ``calls``, replayed in turn."""
    import torch
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for f in calls:
            f()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(reps):
            for f in calls:
                f()
    return min(wall(g.replay, 10) for _ in range(3)) / reps / len(calls)


def rates():
    import torch
    x = torch.zeros(1 << 30, device='cuda')
    y = torch.empty_like(x)
    us = wall(lambda: y.copy_(x), 20)
    print('copy of 4 GiB: %.0f us, %.2f TB/s read and written' % (us, 2 * x.numel() * 4 / us / 1e6), flush=True)
    del x, y
    for kind in (torch.bfloat16, torch.float32):
        a = torch.randn(8192, 8192, device='cuda').to(kind)
        b = torch.randn(8192, 8192, device='cuda').to(kind)
        us = wall(lambda: a @ b, 20)
        print('product of 8192^3 in %s: %.0f us, %.0f TFLOP/s' % (kind, us, 2 * 8192 ** 3 / us / 1e6), flush=True)


def passes(m, case):
    """SETS calls of the case, each with its own data."""
    states = [m.prepare(case, k) for k in range(SETS)]
    if case['op'] == 'adamw':
        return [lambda s=s: m.run(s) for s in states]

    def one(s):                                             # (a graph keeps the leaves' gradients of the last pass: none left over)
        r = m.run(s)
        if case['train']:
            for t in (s['x'], s['gamma'], s['beta']):
                t.grad = None
        return r
    return [lambda s=s: one(s) for s in states]


def table_of_cases():
    import torch
    m = cases()
    for case in m.listed():
        w = m.work(case)['bytes']
        calls = passes(m, case)
        turn = iter(range(1 << 30))
        eager = min(wall(lambda: calls[next(turn) % SETS](), 60) for _ in range(3))
        us = graph_us(calls)
        print('%-18s pass %7.1f us   graph %7.1f us, %5.2f TB/s of %9.2f MB' % (case['name'], eager, us, w / us / 1e6, w / 1e6), flush=True)
        del calls
        torch.cuda.empty_cache()


LN = [(12289, 2048, 'float32'), (16384, 4096, 'bfloat16'), (98304, 32, 'float32'), (6144, 768, 'bfloat16'), (100000, 256, 'float32'),
      (30000, 1024, 'float32'), (60000, 513, 'bfloat16'), (2000, 16384, 'bfloat16'), (16, 768, 'bfloat16'), (70001, 3, 'float32'),
      (100000, 7, 'bfloat16')]
ADAMW = [(n, bits, clip) for bits in (32, 8) for n in (20000, 100000, 200000, 1000000, 3000000, 10000000, 28500000) for clip in (False,)] + \
        [(63600000, 32, True), (3300000, 8, True)]


def table_of_kernels():
    import torch
    from advmix_amd._lib import call, lib
    from advmix_amd.utils.utils import FlatAdamW
    P = lambda t: None if t is None else t.data_ptr()          # noqa: E731
    st = lambda: torch.cuda.current_stream().cuda_stream          # noqa: E731
    for rows, C, name in LN:
        kind, code = getattr(torch, name), {'float32': 0, 'bfloat16': 1, 'float16': 2}[name]
        sets = []
        for k in range(SETS):
            g = torch.Generator(device='cuda').manual_seed(k)
            x, dy = (torch.randn(rows, C, device='cuda', generator=g).to(kind) for _ in range(2))
            part = torch.empty(lib.advmix_layer_norm_parts(rows, C, code) * 2 * C, device='cuda')
            sets.append([x, dy, torch.empty_like(x), torch.empty_like(x), torch.empty(2, rows, device='cuda'), torch.ones(2, C, device='cuda'),
                         torch.zeros(2, C, device='cuda'), part])

        def fwd(s):
            x, _, y, _, stats, par, _, _ = s
            call('advmix_layer_norm_fwd', P(x), C, P(par[0]), P(par[1]), P(y), P(stats[0]), P(stats[1]), rows, C, code, 1e-5, st())

        def bwd(s, sums):
            x, dy, _, dx, stats, par, grad, part = s
            call('advmix_layer_norm_bwd', P(dy), C, P(x), C, P(par[0]), P(stats[0]), P(stats[1]), P(dx), P(grad[0]) if sums else None,
                 P(grad[1]) if sums else None, P(part) if sums else None, 0, rows, C, code, st())
        n = rows * C * sets[0][0].element_size()
        f, b, d = (graph_us([lambda s=s: call_(s) for s in sets]) for call_ in (fwd, lambda s: bwd(s, True), lambda s: bwd(s, False)))
        both = graph_us([lambda s=s: (fwd(s), bwd(s, True)) for s in sets])
        print('layer norm %6d x %5d %-8s forward %6.1f us %5.2f TB/s   backward with its fold %6.1f us %5.2f TB/s   dx alone %6.1f us   both %6.1f us'
              % (rows, C, name, f, 2 * n / f / 1e6, b, 3 * n / b / 1e6, d, both), flush=True)
        del sets
        torch.cuda.empty_cache()
    for n, bits, clip in ADAMW:
        opts = []
        for k in range(SETS):
            cut = [n // 30] * 29
            ps = [torch.nn.Parameter(torch.randn(s, device='cuda')) for s in cut + [n - sum(cut)]]
            o = FlatAdamW([dict(params=ps[:15]), dict(params=ps[15:], weight_decay=0.0)], state_bits=bits, max_norm=1.0 if clip else None)
            o.flat_grads.normal_()
            opts.append(o)
        us = graph_us([o.step for o in opts])
        line = 'AdamW %8d elements in 30 tensors, %2d bits%s %7.1f us %5.2f TB/s' % (
            n, bits, ', clipped' if clip else '', us, n * ((28 if bits == 32 else 16) + (4 if clip else 0)) / us / 1e6)
        if clip:
            norm = graph_us([lambda o=o: call('advmix_grad_sumsq', *o._norm_args, st()) for o in opts])
            line += '   its norm alone %.1f us %.2f TB/s' % (norm, n * 4 / norm / 1e6)
        print(line, flush=True)
        del opts, o, ps
        torch.cuda.empty_cache()


def run_passes(n):
    import torch
    m = cases()
    for case in m.listed():
        calls = passes(m, case)
        for k in range(n):
            calls[k % SETS]()
        torch.cuda.synchronize()
        print(case['name'], flush=True)
        del calls
        torch.cuda.empty_cache()


def kernel_table(where):
    def short(name):
        return re.sub(r'\(anonymous namespace\)::|void ', '', name).split('(')[0]

    def rows(what, kind):
        for f in sorted(glob.glob(os.path.join(where, '**', what + '_' + kind + '.csv'), recursive=True)):
            with open(f) as fh:
                yield from (r for r in csv.DictReader(fh) if any(k in r['Kernel_Name'] for k in OURS))
    times, counts = {}, {'fetch': {}, 'write': {}}
    for r in rows('time', 'kernel_trace'):
        at = (short(r['Kernel_Name']), int(r['Grid_Size_X']) * int(r['Grid_Size_Y']))
        times.setdefault(at, []).append((int(r['End_Timestamp']) - int(r['Start_Timestamp'])) / 1e3)
    for what, into in counts.items():
        for r in rows(what, 'counter_collection'):
            into.setdefault((short(r['Kernel_Name']), int(r['Grid_Size'])), []).append(float(r['Counter_Value']))
    print('kernel,grid_threads,launches,median_us,min_us,fetch_MiB,write_MiB')
    for at, t in times.items():
        got = ['%.2f' % (statistics.median(c[at]) / 1024) if at in c else '' for c in counts.values()]
        print('"%s",%d,%d,%.2f,%.2f,%s,%s' % (at[0], at[1], len(t), statistics.median(t), min(t), *got))


if __name__ == '__main__':
    how = sys.argv[1] if len(sys.argv) > 1 else ''
    if how == '--table':
        kernel_table(sys.argv[2])
    elif how == '--passes':
        run_passes(int(sys.argv[2]))
    elif how == '--kernels':
        table_of_kernels()
    elif how == '':
        rates()
        table_of_cases()
    else:
        sys.exit(__doc__)

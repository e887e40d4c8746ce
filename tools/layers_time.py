#!/usr/bin/env python3
"""Times of layer norm, dropout and decay attention: the cases of perf/operators.py and more sizes of the same operators.

    python3 tools/layers_time.py time [--plain] [NAME ..]      time of a pass, us: median and least of 9 batches of 10 passes
    rocprofv3 -M --kernel-trace -d DIR -o p -f csv -- python3 tools/layers_time.py run [NAME ..]      20 passes of each
    python3 tools/layers_time.py stats DIR/p_kernel_trace.csv OUT.csv [NAME ..]      kernel times, case by case
    rocprofv3 -M --pmc COUNTERS -d DIR -o p -f csv -- python3 tools/layers_time.py once NAME      3 passes
    python3 tools/layers_time.py counters OUT.json TITLE DIR/p_counter_collection.csv ..       the last pass's counters, added to OUT

NAME: part of a case's name (default: all of them).  -M leaves kernel names as the linker has them, which `stats` and `counters`
read: taken apart by the profiler, those with 16-bit types come out wrong."""
import collections
import csv
import json
import os
import re
import statistics
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def cases():
  import torch
  from perf import operators
  operators.DTYPES.setdefault('f16', torch.float16)
  more = []

  def attn(T, N, H, dk, dv, dtype, train, cuts=0.005, ragged=False):
    more.append(dict(name='attn %d x %d x %d heads of %d / %d %s %s' % (T, N, H, dk, dv, dtype, 'train' if train else 'fwd'),
                     op='decay_attention', T=T, N=N, H=H, dk=dk, dv=dv, dtype=dtype, cuts=cuts, ragged=ragged, train=train))

  for dtype in ('f32', 'bf16', 'f16'):
    for train in (False, True):
      attn(256, 512, 4, 64, 64, dtype, train)
  for dtype in ('f32', 'bf16'):
    for d in (16, 32, 80, 96, 128):
      attn(128, 512, 4, d, d, dtype, True)
  attn(25, 1615, 8, 98, 67, 'bf16', True)
  for rows, width, dtype in ((1 << 20, 32, 'f32'), (1 << 18, 128, 'bf16'), (65536, 1024, 'bf16'), (1 << 18, 257, 'f32'),
                             (1 << 18, 257, 'bf16'), (1 << 18, 260, 'f32'), (1 << 18, 264, 'bf16'), (4096, 8192, 'bf16'),
                             (4096, 12000, 'bf16')):
    more.append(dict(name='norm %d x %d %s train' % (rows, width, dtype), op='layer_norm', rows=rows, width=width, dtype=dtype,
                     relu=False, train=True))
  for N, d in ((65536, 16), (262144, 8), (1024, 128)):
    more.append(dict(name='step %d envs x 4 heads of %d' % (N, d), op='decay_step', N=N, H=4, dk=d, dv=d, dtype='f32', cuts=0.005))
  return operators, operators.listed() + more


def chosen(names):
  operators, all_cases = cases()
  return operators, [c for c in all_cases if not names or any(n in c['name'] for n in names)]


def passes(names, own, count):
  import torch
  operators, some = chosen(names)
  operators.own = own
  for case in some:
    state = operators.prepare(case, 1)
    for _ in range(count):
      operators.run(state)
    torch.cuda.synchronize()
    yield operators, case, state


def time_cases(names, own):
  import torch
  for operators, case, state in passes(names, own, 3):
    times = []
    for _ in range(9):
      a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
      a.record()
      for _ in range(10):
        operators.run(state)
      b.record()
      b.synchronize()
      times.append(a.elapsed_time(b) * 100)
    work = operators.work(case)
    t = statistics.median(times)
    print('%-48s %10.1f us, least %10.1f   %6.2f TB/s %7.1f TFLOP/s' % (
        case['name'], t, min(times), work['bytes'] / t / 1e6, work['flops'] / t / 1e6), flush=True)


KERNEL = re.compile(r'k_(norm|dropout|scan|join|step|next)')


def kernel_name(name):
  m = re.search(r'(k_(?:norm|dropout|scan|step)\w*?)I(DF16b|DF16_|f)((?:L[ib]\d+E)+)E', name)
  if m:
    kind = {'DF16b': 'bf16', 'DF16_': 'f16', 'f': 'float'}[m[2]]
    args = [v if t == 'i' else ('false', 'true')[int(v)] for t, v in re.findall(r'L([ib])(\d+)E', m[3])]
    return '%s<%s>' % (m[1], ', '.join([kind] + args))
  return re.search(r'k_(norm_fold|join|next_call)|$', name)[0] or name


def stats(trace, out, *names):
  """A case's inputs come from torch's random kernels: what follows on some of those is the next case."""
  labels = [c['name'] for c in chosen(names)[1]]
  rows, at, between = collections.OrderedDict(), -1, True
  for r in sorted(csv.DictReader(open(trace)), key=lambda r: int(r['Start_Timestamp'])):
    between |= 'distribution' in r['Kernel_Name']
    if KERNEL.search(r['Kernel_Name']):
      at, between = at + between, False
      grid = 'x'.join(str(int(r['Grid_Size_' + d]) // int(r['Workgroup_Size_' + d])) for d in 'XYZ')
      key = (labels[at], kernel_name(r['Kernel_Name']), grid, r['Workgroup_Size_X'], r['Scratch_Size'])
      rows.setdefault(key, []).append((int(r['End_Timestamp']) - int(r['Start_Timestamp'])) / 1e3)
  with open(out, 'w') as f:
    f.write('case,kernel,workgroups,threads,scratch_bytes,calls,median_us,min_us\n')
    for key, t in rows.items():
      f.write('"%s","%s",%s,%s,%s,%d,%.1f,%.1f\n' % (*key, len(t), statistics.median(t), min(t)))


def counters(out, title, files):
  res = json.load(open(out)) if os.path.exists(out) else {}
  mine = res[title] = {}
  for name in files:
    for r in csv.DictReader(open(name)):
      if KERNEL.search(r['Kernel_Name']):
        key = '%s, %d workgroups' % (kernel_name(r['Kernel_Name']), int(r['Grid_Size']) // int(r['Workgroup_Size']))
        mine.setdefault(key, {})[r['Counter_Name']] = float(r['Counter_Value'])
  json.dump(res, open(out, 'w'), indent=1)


def main():
  what, args = sys.argv[1], sys.argv[2:]
  if what == 'time':
    time_cases([a for a in args if a != '--plain'], '--plain' not in args)
  elif what in ('run', 'once'):
    for _, case, _ in passes(args, True, 20 if what == 'run' else 3):
      print(case['name'], flush=True)
  elif what == 'stats':
    stats(*args)
  else:
    counters(args[0], args[1], args[2:])


if __name__ == '__main__':
  main()

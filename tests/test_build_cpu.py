"""CPU: what the build looks at: no kernel spills vector registers, and every source of the folder is one that is built."""
import os
import re
import subprocess
import sys

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'text-style-transfer_amd', 'csrc')

REPORT = """unit.hip:10:1: remark: Function Name: kernel_a [-Rpass-analysis=kernel-resource-usage]
   10 | __global__ void kernel_a() {
unit.hip:10:1: remark:     VGPRs: 256 [-Rpass-analysis=kernel-resource-usage]
unit.hip:10:1: remark:     ScratchSize [bytes/lane]: 0 [-Rpass-analysis=kernel-resource-usage]
unit.hip:10:1: remark:     SGPRs Spill: 6 [-Rpass-analysis=kernel-resource-usage]
unit.hip:10:1: remark:     VGPRs Spill: 0 [-Rpass-analysis=kernel-resource-usage]
unit.hip:20:1: remark: Function Name: kernel_b [-Rpass-analysis=kernel-resource-usage]
unit.hip:20:1: remark:     ScratchSize [bytes/lane]: 0 [-Rpass-analysis=kernel-resource-usage]
unit.hip:20:1: remark:     VGPRs Spill: 0 [-Rpass-analysis=kernel-resource-usage]
"""


def check(report):
    return subprocess.run([sys.executable, os.path.join(CSRC, 'check_spills.py'), 'unit'], input=report, capture_output=True, text=True)


def test_a_kernel_that_spills_vector_registers_fails_the_build():
    assert check(REPORT).returncode == 0 and check('').returncode == 0
    head, tail = REPORT.rsplit('VGPRs Spill: 0', 1)
    for bad in (head + 'VGPRs Spill: 12' + tail, REPORT.replace('lane]: 0', 'lane]: 48')):
        r = check(bad)
        assert r.returncode == 1 and 'kernel_b' in r.stderr
    with open(os.path.join(CSRC, 'build.sh')) as f:
        assert re.search(r'python3 check_spills.py \$1 < \S+ \|\| return 1', f.read())


def test_every_source_is_built():
    """A kernel source that no build names is a stale copy of one that is."""
    with open(os.path.join(CSRC, 'build.sh')) as f:
        text = f.read()
    units = re.search(r'^UNITS="([^"]+)"', text, re.M).group(1).split()
    kept = subprocess.run(['git', 'ls-files', '--', '.'], cwd=CSRC, capture_output=True, text=True)
    files = kept.stdout.split() if kept.returncode == 0 and kept.stdout else os.listdir(CSRC)
    assert sorted(n[:-4] for n in files if n.endswith('.hip')) == sorted(units)
    assert [n for n in files if n.endswith('.cpp')] == ['calls.cpp'] and 'calls.cpp' in text


def test_the_calls_module_is_for_this_torch():
    import types

    import pytest
    import torch
    from tst_amd import _lib
    assert _lib.calls.built_for == torch.__version__.split('+')[0]
    _lib._check_calls(_lib.calls)
    for other in (types.SimpleNamespace(built_for='1.0.0'), types.SimpleNamespace()):
        with pytest.raises(ImportError, match='build it with'):
            _lib._check_calls(other)

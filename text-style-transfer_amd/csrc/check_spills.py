"""Reads a compile job's kernel resource report (stdin) and fails if a kernel keeps vector registers in memory.

    hipcc ... -Rpass-analysis=kernel-resource-usage -c unit.hip 2> report; python3 check_spills.py unit < report

A prompt attention kernel that spilled, compiled with matrix results in ordinary registers, gave wrong values, and nothing in its source showed
why; no kernel of this library needs to spill, so none may.  (Scalar registers kept in lanes of vector registers are not meant: several kernels
have some.)
"""
import re
import sys


def spilled(report):
    """(kernels in the report, [(kernel, what, how much)] of those that spill vector registers or use scratch memory)"""
    name, kernels, bad = None, 0, []
    for line in report.splitlines():
        m = re.search(r'remark:\s+([^:]+): (\S+)', line)
        if m is None:
            continue
        key, value = m.groups()
        if key == 'Function Name':
            name, kernels = value, kernels + 1
        elif (key == 'VGPRs Spill' or key.startswith('ScratchSize')) and value != '0':
            bad.append((name, key, value))
    return kernels, bad


if __name__ == '__main__':
    _, bad = spilled(sys.stdin.read())
    for name, key, value in bad:
        print('%s: %s has %s: %s' % (sys.argv[1], name, key, value), file=sys.stderr)
    sys.exit(1 if bad else 0)

"""Build-time guards of the product's hand-counted loops (CPU only): the ring and streaming kernels of csrc/fp8_gemm.h feed LDS by inline-asm
LDS-DMA that hipcc's bookkeeping does not see and wait for it with counted vmcnt(2 groups).  A spill, a hoisted load or a wait that hipcc
adds by itself inside the steps would turn that into a race or a stall."""
import os
import re
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, 'tools'))
import check_loops as C  # noqa: E402


@pytest.fixture(scope='module')
def kernels():
    """{mangled name: (instructions, resource remarks)} of the product's kernels."""
    s_path, r_path = C.build_asm('fp8')
    res, cur = {}, None
    for line in open(r_path):
        m = re.search(r'Function Name: (\S+)', line)
        if m:
            cur = res.setdefault(m.group(1), {})
            continue
        m = re.search(r'remark: (?:\S+: )?\s*([A-Za-z ]+?)(?: \[[^\]]*\])?: (\d+)', line)
        if m and cur is not None:
            cur[m.group(1).strip()] = int(m.group(2))
    return {k: (v, res.get(k, {})) for k, v in C.functions(s_path).items() if 'fp8_gemm' in k}


def _steady(lines):
    """Instruction mix of the basic block with the most LDS-DMA among those that multiply inside the loop (two steps)."""
    marks = [i for i, l in enumerate(lines) if re.match(r'^\.LBB', l)] + [len(lines)]
    best = None
    for a, b in zip(marks, marks[1:]):
        m = C.mix(lines, (a, b - 1))
        if m.get('mfma') and m.get('lds_dma') and m.get('barrier') == 2:
            assert best is None, "two loop bodies"
            best = m
    return best


def _tile(name):
    if 'stream' in name:
        return 4, 4
    m = re.search(r'Li(\d)ELi(\d)E', name)
    return int(m.group(1)), int(m.group(2))


def test_no_product_kernel_spills(kernels):
    assert len(kernels) >= 15
    for name, (_, r) in kernels.items():
        assert r and r.get('VGPRs Spill', 0) == 0 and r.get('ScratchSize', 0) == 0, (name, r)


def test_steps_hold_what_their_waits_count(kernels):
    seen = 0
    for name, (lines, r) in kernels.items():
        if 'ring' not in name and 'stream' not in name:
            continue
        ni, nj = _tile(name)
        q = ni + nj
        half = 'IDF16' in name
        want = {'mfma': 2 * ni * nj * (1 if half else 4), 'lds_dma': 2 * q, 'barrier': 2, 'vmcnt_waits': {2 * q: 2}, 'ds_read': 4 * q + q}
        assert _steady(lines) == want, (name, _steady(lines), want)
        if ni * nj == 16:
            assert r['AGPRs'] == 256, (name, r)
        seen += 1
    assert seen >= 8 + 2


def test_results_leave_the_accumulators_behind_the_padding(kernels):
    """The streaming kernel reads its accumulators by asm, for which hipcc pads nothing: the first read stands behind two s_nop 15."""
    for name, (lines, _) in kernels.items():
        if 'stream' not in name:
            continue
        ops = [l.strip() for l in lines if l.strip() and not l.strip().startswith((';', '.'))]
        last = max(i for i, l in enumerate(ops) if l.startswith('v_mfma'))
        nops = [i for i, l in enumerate(ops) if l.startswith('s_nop 15') and i > last]
        reads = [i for i, l in enumerate(ops) if l.startswith('v_accvgpr_read') and i > last]
        assert len(nops) >= 2 and reads and reads[0] > nops[1], (name, nops[:3], reads[:3], last)
        assert not [i for i, l in enumerate(ops) if l.startswith('v_accvgpr_read') and i < last], name

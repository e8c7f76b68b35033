"""The rule of test_asm_hazards.py on the grouped products' kernels (CPU only): no instruction may
touch a pending inline-assembly read's destination, and no branch may leave with one pending, before
the next ``s_waitcnt lgkmcnt(0)``."""
import re

import pytest

from test_asm_hazards import HIPCC, _assembly, _violations

pytestmark = pytest.mark.skipif(HIPCC is None, reason="hipcc not available")


def _grouped_kernels(text: str) -> dict[str, list[str]]:
    bodies, name = {}, None
    for line in text.splitlines():
        m = re.match(r"^(_ZN2ws\w*grouped_(?:fast|ring|grad_fast|grad_ring)_kernel\w*):", line)
        if m:
            name = m.group(1)
            bodies[name] = []
        elif name is not None:
            if line.startswith(".Lfunc_end"):
                name = None
            else:
                bodies[name].append(line)
    return bodies


def test_fragment_reads_are_waited_for_before_use(tmp_path):
    kernels = _grouped_kernels(_assembly("grouped.hip", tmp_path))
    # 256 x 256 tiles in two layouts, four smaller tiles in each, three of them in slices too; gradients in two
    # types on all five.
    assert len(kernels) == 2 + 8 + 6 + 2 + 8, sorted(kernels)
    for name, body in kernels.items():
        reads, bad = _violations(body)
        # The smaller tiles' K-contiguous fragments are read by the compiler.
        assert reads > 0 or ("grouped_ring" in name and re.search(r"Li0ELb[01]EEEvNS_13GroupedParamsE$", name)), name
        assert not bad, (name, bad[:5])

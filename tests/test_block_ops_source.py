"""Rules that the sources of overlapping kernels keep, which no run of them can show."""
import re
from pathlib import Path

KERNELS = Path(__file__).resolve().parent.parent / "parameter_server_b200" / "csrc" / "kernels"


def test_launches_that_overlap_their_predecessor_read_coherently():
    """A non-coherent load is defined only for memory that nothing writes while the kernel runs; a kernel that may begin before its
    predecessor has ended, or that puts its result in its input's place, has no such memory."""
    for name in ("linear_fused.cuh", "linear_few.cuh", "act8_wgrad.cu"):
        text = (KERNELS / name).read_text()
        assert "start_early()" in text or "launch_pairs(" in text
        assert not re.search(r"ld_nc|ld\.global\.nc|__ldg\(|__restrict__", text), name

"""What bench.py reports from committed files, without a GPU."""
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import bench  # noqa: E402


@pytest.mark.parametrize("path,kernel", [
    (bench.TRAFFIC_FILE, "k_gemv2_q4k"), (bench.SKINNY_TRAFFIC_FILE, "k_gemv_mma_q4k_rec"),
    (bench.CV2_TRAFFIC_FILE, "k_gemv2_q80"), (bench.Q80_TRAFFIC_FILE, "k_gemv2_q80")])
def test_counter_summaries_are_of_these_sources(path, kernel):
    """The HBM bytes a launch that the roofline line reports: their summary was measured on the kernel
    sources of this tree (else the line reports none)."""
    assert bench.measured_traffic(path, kernel) > 0

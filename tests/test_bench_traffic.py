"""CPU test: the step kernel's DRAM traffic that bench.py reports was captured
on the sources in the tree.  Whoever changes those captures it again."""
import bench


def test_the_traffic_figure_belongs_to_the_step_kernels_sources():
    assert bench.kernel_sources_digest() == bench.NCU_TRAFFIC_DIGEST
    assert bench.measured_traffic_per_step() == bench.NCU_TRAFFIC_PER_STEP

"""append_block_scaled where the warps of one CTA hold K jobs, V jobs and none at the same time, several warps to a
job: they meet at one barrier, and the codes and scales are the defined bits."""
import pytest

from test_block_scaled_append_gpu import compare, make, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["int8", "e5m2"])
@pytest.mark.parametrize("hk,d,bs,rotary", [(1, 128, 64, 128), (3, 128, 64, 64), (3, 64, 128, 64), (5, 128, 128, 32),
                                            (1, 256, 64, 256), (7, 64, 64, 16), (3, 512, 32, 512)])
def test_odd_heads_and_several_warps_to_a_job(cuda_device, cache, hk, d, bs, rotary):
    """K is rotated, V is not; new rows that fill, begin, end in and pass over blocks."""
    c = make(hk * d + bs, [0, 50, 3, 127, 0], [300, 200, 131, 129, 64], hk, d, bs, cache, rotary, 2)
    compare(run(c, cuda_device), reference(c))


def test_infinities_in_some_warps_only(cuda_device):
    """One warp of a job takes the careful way, its neighbours the usual one."""
    c = make(3, [0, 20], [128, 200], 3, 128, 64, "e4m3", 128, 2)
    for row in (5, 70, 130, 131, 300):
        c["k"][row, row % 3, row % 128] = float("inf") if row % 2 else float("nan")
        c["v"][row + 1, row % 3, row % 128] = -float("inf")
    compare(run(c, cuda_device), reference(c))
